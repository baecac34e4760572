"""The 4-bit cache operators and packed prompt attention, as they are measured.

Three operators that one serving step uses in turn:

  append   RoPE of a step's queries and keys and the store of its keys and
           values into a paged cache that holds them in 4 bits
  decode   attention of single tokens over that cache
  packed   causal attention of whole prompts of different lengths, packed row
           after row, with grouped heads

`run` computes them in their plain form, in elementary torch operations in 32
bits, or (with `own` set) through libfish.so's entry points.

The cache's format. Keys and values of one position and kv head are cut into
groups of 32 dimensions. A group holds lo = f16(min) and d = f16((max - lo) /
15), min and max clamped to the f16 range, and per value the 4-bit code
rint((x - lo) * (1 / d)) clamped to 0..15 (code 0 where d = 0); it stands for
lo + d * code. A page holds 16 positions of every layer; inside a layer each kv
head has one record
  K codes [16][D/2]  K d [16][GP] f16  K lo [16][GP] f16  and the same for V,
GP = D / 32 rounded up to even. A row's K byte for dimension 32 g + 8 t + n is
4 GP' t + 4 g + n / 2 (GP' = D / 32), its V byte for dimension 32 g + 4 h + n
is 2 GP' h' + 2 g + n / 2 with h' = h, or h ^ 4 in rows where bit 1 of the
position is set; even n take the low nibble.
"""
import math

import torch

own = False

TYPES = {"f32": (0, torch.float32), "f16": (1, torch.float16), "bf16": (30, torch.bfloat16)}
PAGE = 16


# ------------------------------------------------------------------- the cases

def listed():
    def append(name, **k):
        return {"name": name, "op": "append", "layers": 1, **k}

    def decode(name, **k):
        return {"name": name, "op": "decode", "softcap": 0.0, "window": 0, **k}

    def packed(name, **k):
        return {"name": name, "op": "packed", "softcap": 0.0, "window": 0, **k}

    return [
        # one session's next token on the 8B shape, f32 as the engine's activations are: latency
        append("append 1 token f32", T=1, seqs=1, H=32, HKV=8, D=128, rot=128, neox=False, type="f32", out="f32"),
        # a batch of 64 sessions, one token each, the 7B shape
        append("append 64 sessions f16", T=64, seqs=64, H=28, HKV=4, D=128, rot=128, neox=True, type="f16", out="f16"),
        # an odd run of prompt tokens, head dimension 96, a partial rotation, f32 in and f16 out
        append("append 777 tokens d96", T=777, seqs=3, H=12, HKV=4, D=96, rot=64, neox=True, type="f32", out="f16"),
        # whole prompts of a batch on the 70B shape: bandwidth
        append("append 16384 tokens bf16", T=16384, seqs=8, H=64, HKV=8, D=128, rot=128, neox=False, type="bf16",
               out="bf16"),
        # one session's next token after a short chat: latency
        decode("decode 1 x 577 f32", T=1, low=577, high=577, H=32, HKV=8, D=128, type="f32"),
        # one session over a whole book
        decode("decode 1 x 131071 bf16", T=1, low=131071, high=131071, H=64, HKV=8, D=128, type="bf16"),
        # 64 sessions a little past a 2048-token document
        decode("decode 64 x 2100 f16", T=64, low=2049, high=2180, H=28, HKV=4, D=128, type="f16"),
        # batch 32 after 4096-token prompts and answers of different lengths, the 70B shape
        decode("decode 32 x 4600 bf16", T=32, low=4097, high=5100, H=64, HKV=8, D=128, type="bf16"),
        # one chat prompt, the 8B shape
        packed("packed 1 x 512 bf16", seqs=1, low=512, high=512, H=32, HKV=8, D=128, type="bf16"),
        # many short requests, a head dimension of 64, every length from none on
        packed("packed 64 x 0-300 f16", seqs=64, low=0, high=300, H=8, HKV=8, D=64, type="f16"),
        # a batch of documents of different lengths, the 7B shape
        packed("packed 16 x 100-2047 f16", seqs=16, low=100, high=2047, H=28, HKV=4, D=128, type="f16"),
        # one long prompt on the 70B shape: the tensor cores' rate
        packed("packed 1 x 16384 bf16", seqs=1, low=16384, high=16384, H=64, HKV=8, D=128, type="bf16"),
    ]


def _log_int(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    HKV = rng.choice([1, 2, 4, 8])
    H = HKV * rng.choice([1, 2, 3, 4, 5, 7, 8])
    c = {"op": rng.choice(["append", "decode", "packed"]), "H": H, "HKV": HKV, "D": rng.choice([64, 96, 128, 128]),
         "type": rng.choice(["f16", "bf16"])}
    if c["op"] == "append":
        c["type"] = rng.choice(["f32", "f16", "bf16"])
        T = _log_int(rng, 1, 9000)
        c.update(T=T, seqs=rng.randint(1, min(T, 16)), layers=rng.choice([1, 1, 2]), neox=rng.random() < 0.5,
                 rot=rng.choice([c["D"], c["D"], c["D"] // 2]), out=rng.choice([c["type"], "f16", "bf16"]))
        return c
    c["softcap"] = rng.choice([0.0, 0.0, 0.0, 50.0])
    c["window"] = rng.choice([0, 0, 0, 1000])
    if c["op"] == "decode":
        c["type"] = rng.choice(["f32", "f16", "bf16"])
        T = _log_int(rng, 1, 64)
        c.update(T=T, high=_log_int(rng, 1, min(131071, 200000 // T)))
        c["low"] = rng.randint(1, c["high"])
        return c
    c["seqs"] = _log_int(rng, 1, 64)
    c["high"] = _log_int(rng, 1, 30000 // c["seqs"] if c["seqs"] > 2 else 9000)
    c["low"] = rng.randint(0, c["high"])
    return c


def _lengths(case, count):
    """`count` lengths from low to high, the same for every seed: the work of a case is its own."""
    span = case["high"] - case["low"]
    return [case["low"] + (span * ((7 * i + 3) % count)) // max(1, count - 1) if count > 1 else case["high"]
            for i in range(count)]


def _record(D):
    """Bytes of one kv head's record in a page, and of its parts: codes, one scale array."""
    codes, scales = PAGE * D // 2, PAGE * 2 * _gp(D)
    return 2 * (codes + 2 * scales), codes, scales


def _gp(D):
    return (D // 32 + 1) // 2 * 2


def work(case):
    H, HKV, D = case["H"], case["HKV"], case["D"]
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "append":
        T, vals = case["T"], (H + 2 * HKV) * D
        out = 4 if case["out"] == "f32" else 2
        return {"bytes": T * (vals * (size + out) + HKV * _record(D)[0] // PAGE + case["rot"] * 4 + 8),
                "flops": T * (3 * (H + HKV) * case["rot"] + 8 * HKV * D)}
    if case["op"] == "decode":
        T, lens = case["T"], _lengths(case, case["T"])
        seen = sum(min(n, case["window"] or n) for n in lens)
        return {"bytes": seen * HKV * _record(D)[0] // PAGE + 2 * T * H * D * size + seen // 4 + 8 * T,
                "flops": 4 * seen * H * D}
    lens, w = _lengths(case, case["seqs"]), case["window"]
    pairs = sum(n * (n + 1) // 2 - (max(0, n - w) * (n - w + 1) // 2 if w and n > w else 0) for n in lens)
    return {"bytes": sum(lens) * (2 * H + 2 * HKV) * D * size + 4 * (case["seqs"] + 1) + 16, "flops": 4 * pairs * H * D + 1}


# ------------------------------------------------------------------ the inputs

def _normal(shape, dtype, gen):
    """Values as projections give them: unit normals, a few dimensions with a larger spread."""
    x = torch.randn(shape, device="cuda", generator=gen)
    spread = torch.exp(0.4 * torch.randn(shape[-1:], device="cuda", generator=gen))
    return (x * spread).to(dtype)


def _tables(n, rot):
    """cos and sin of position * 500000^(-2 i / rot), formed in 64 bits."""
    f = torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot
    a = torch.arange(n, device="cuda", dtype=torch.float64)[:, None] * torch.pow(500000.0, -f)[None, :]
    return a.cos().float().contiguous(), a.sin().float().contiguous()


def _pages(lens, layers, HKV, D, gen):
    """A pool of pages in random order and the page tables of sequences of these lengths."""
    each = [(n + PAGE - 1) // PAGE for n in lens]
    n_pages, stride = sum(each) + 3, max(each) + 1
    order = torch.randperm(n_pages, device="cuda", generator=gen).to(torch.int32)
    at = torch.tensor([sum(each[:i]) for i in range(len(each))], device="cuda")
    index = at[:, None] + torch.arange(stride, device="cuda")[None, :]
    table = order[index.clamp(max=n_pages - 1)].contiguous()
    pool = torch.zeros(n_pages * layers * HKV * _record(D)[0], dtype=torch.uint8, device="cuda")
    return pool, table


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    H, HKV, D = case["H"], case["HKV"], case["D"]
    dtype = TYPES[case["type"]][1]
    s = dict(case)
    if case["op"] == "append":
        T, n = case["T"], case["seqs"]
        lens = [T // n + (i < T % n) for i in range(n)]
        start = [(37 * i + 5) % 50 if T > n else 100 + 61 * i for i in range(n)]  # a chunk after what was there, or one token
        s["seq"] = torch.cat([torch.full((m,), i, dtype=torch.int32, device="cuda") for i, m in enumerate(lens)])
        s["pos"] = torch.cat([torch.arange(p, p + m, dtype=torch.int32, device="cuda") for p, m in zip(start, lens)])
        s["layer"] = case["layers"] - 1
        s["pool"], s["table"] = _pages([p + m for p, m in zip(start, lens)], case["layers"], HKV, D, gen)
        s["cos"], s["sin"] = _tables(max(p + m for p, m in zip(start, lens)), case["rot"])
        # the three projections as one matrix product leaves them: a row is q | k | v
        s["qkv"] = _normal((T, (H + 2 * HKV) * D), dtype, gen)
        for name, width in (("q_out", H * D), ("k_out", HKV * D), ("v_out", HKV * D)):
            s[name] = torch.empty((T, width), dtype=TYPES[case["out"]][1], device="cuda")
    elif case["op"] == "decode":
        T, lens = case["T"], _lengths(case, case["T"])
        s["layers"], s["layer"] = 1, 0
        s["pool"], s["table"] = _pages(lens, 1, HKV, D, gen)
        s["seq"] = torch.arange(T, dtype=torch.int32, device="cuda")
        s["pos"] = torch.tensor([n - 1 for n in lens], dtype=torch.int32, device="cuda")
        s["keys"] = max(lens)
        seq = torch.cat([torch.full((n,), i, device="cuda") for i, n in enumerate(lens)])
        pos = torch.cat([torch.arange(n, device="cuda") for n in lens])
        k, v = (_normal((len(pos), HKV, D), torch.float32, gen) for _ in range(2))
        _store(s, s["table"][seq, pos // PAGE].long(), pos % PAGE, k, v)
        s["q"] = _normal((T, H * D), dtype, gen)
        s["result"] = torch.empty_like(s["q"])
    else:
        s["lens"] = _lengths(case, case["seqs"])
        N = max(1, sum(s["lens"]))
        s["cu"] = torch.tensor([sum(s["lens"][:i]) for i in range(len(s["lens"]) + 1)], dtype=torch.int32, device="cuda")
        s["q"], s["k"], s["v"] = (_normal((N, h * D), dtype, gen) for h in (H, HKV, HKV))
        s["result"] = torch.zeros_like(s["q"])
    if own:
        _plan(s)
    return s


# -------------------------------------------------------------- the plain forms

def _rotate(x, cos, sin, rot, neox):
    """x [T][heads][D] in 32 bits, rotated for its tokens' table rows [T][rot / 2]."""
    a, b = (x[..., :rot // 2], x[..., rot // 2:rot]) if neox else (x[..., 0:rot:2], x[..., 1:rot:2])
    cos, sin = cos[:, None, :], sin[:, None, :]
    y0, y1 = a * cos - b * sin, a * sin + b * cos
    y = torch.cat((y0, y1), -1) if neox else torch.stack((y0, y1), -1).flatten(-2)
    return torch.cat((y, x[..., rot:]), -1)


def _quantise(x):
    """Codes [..][groups][32] and the f16 scales of x's groups of 32 values."""
    x = x.unflatten(-1, (-1, 32))
    lo = x.amin(-1).clamp(-65504.0, 65504.0).half()
    hi = x.amax(-1).clamp(-65504.0, 65504.0)
    d = ((hi - lo.float()) / 15.0).half()
    inv = torch.where(d > 0, 1.0 / d.float(), 0.0)
    codes = ((x - lo.float()[..., None]) * inv[..., None]).round().clamp(0, 15)
    return codes, d, lo


def _parts(s):
    """The pool's arrays, each [pages][layers][heads][16][..]: codes in bytes, scales in f16; K's, then V's."""
    D, (rec, codes, scales) = s["D"], _record(s["D"])
    p = s["pool"].view(-1, s["layers"], s["HKV"], rec)
    got, at = [], 0
    for _ in range(2):
        got.append(p[..., at:at + codes].unflatten(-1, (PAGE, D // 2)))
        for k in range(2):
            lo = at + codes + k * scales
            got.append(p[..., lo:lo + scales].view(torch.float16).unflatten(-1, (PAGE, _gp(D))))
        at += codes + 2 * scales
    return got


def _store(s, page, row, k, v):
    """Quantises k and v [T][heads][D] into rows `row` of pages `page`; gives back the values that they then stand for."""
    groups, layer, told = s["D"] // 32, s["layer"], []
    for x, (codes_at, d_at, lo_at), is_v in ((k, _parts(s)[:3], False), (v, _parts(s)[3:], True)):
        codes, d, lo = _quantise(x)
        told.append((lo.float()[..., None] + d.float()[..., None] * codes).flatten(-2))
        c = codes.to(torch.uint8)
        if is_v:  # [heads][group][8][4] to [8][group][4], the halves of the 8 swapped in every second pair of rows
            c = c.unflatten(-1, (8, 4)).transpose(-3, -2)
            c = torch.where(((row // 2) % 2 == 1)[:, None, None, None, None], c.roll(4, -3), c)
        else:  # [heads][group][4][8] to [4][group][8]
            c = c.unflatten(-1, (4, 8)).transpose(-3, -2)
        c = c.flatten(-3)
        codes_at[page, layer, :, row] = c[..., 0::2] | (c[..., 1::2] << 4)
        d_at[page, layer, :, row, :groups] = d
        lo_at[page, layer, :, row, :groups] = lo
    return told


def _values(s, pages):
    """What the pages [..] hold: K and V [..][16][heads][D]."""
    groups, got, parts = s["D"] // 32, [], _parts(s)
    row = torch.arange(PAGE, device="cuda")
    for (codes, d, lo), is_v in ((parts[:3], False), (parts[3:], True)):
        b = codes[pages, s["layer"]]
        c = torch.stack((b & 15, b >> 4), -1).flatten(-2)
        if is_v:
            c = c.unflatten(-1, (8, groups, 4))
            c = torch.where(((row // 2) % 2 == 1)[:, None, None, None], c.roll(4, -3), c)
        else:
            c = c.unflatten(-1, (4, groups, 8))
        c = c.transpose(-3, -2).flatten(-2).float()
        x = lo[pages, s["layer"]][..., :groups, None].float() + d[pages, s["layer"]][..., :groups, None].float() * c
        got.append(x.flatten(-2).transpose(-3, -2))
    return got


def _softmax(score, seen, softcap):
    """Weights of scores [..][keys]; keys that are not seen weigh nothing."""
    if softcap:
        score = softcap * torch.tanh(score / softcap)
    score = torch.where(seen, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    w = torch.exp(score - torch.where(top > -math.inf, top, 0.0))
    total = w.sum(-1, keepdim=True)
    return w / torch.where(total > 0, total, 1.0)


def _append(s):
    H, HKV, D = s["H"], s["HKV"], s["D"]
    pos = s["pos"].long()
    x = s["qkv"].float().unflatten(-1, (-1, D))
    turned = _rotate(x[:, :H + HKV], s["cos"][pos], s["sin"][pos], s["rot"], s["neox"])
    page = s["table"][s["seq"].long(), pos // PAGE].long()
    k, v = _store(s, page, pos % PAGE, turned[:, H:], x[:, H + HKV:])
    out = TYPES[s["out"]][1]
    return {"q": turned[:, :H].flatten(1).to(out), "k": k.flatten(1).to(out), "v": v.flatten(1).to(out), "pool": s["pool"]}


def _decode(s):
    H, HKV, D = s["H"], s["HKV"], s["D"]
    used = (s["keys"] + PAGE - 1) // PAGE
    k, v = _values(s, s["table"][s["seq"].long(), :used].long())
    k, v = (x.flatten(1, 2).transpose(1, 2) for x in (k, v))  # [T][heads][keys][D]
    q = s["q"].float().unflatten(-1, (HKV, H // HKV, D))
    score = q @ k.transpose(-1, -2) * (1.0 / math.sqrt(D))
    key = torch.arange(used * PAGE, device="cuda")[None, :]
    pos = s["pos"].long()[:, None]
    seen = key <= pos
    if s["window"]:
        seen &= key > pos - s["window"]
    return (_softmax(score, seen[:, None, None, :], s["softcap"]) @ v).flatten(1).to(s["q"].dtype)


def _packed(s):
    H, HKV, D = s["H"], s["HKV"], s["D"]
    B, most = len(s["lens"]), max(s["lens"])
    if not most:
        return s["result"]
    cu = s["cu"].long()
    row = cu[:-1, None] + torch.arange(most, device="cuda")[None, :]  # [B][most]
    held = torch.arange(most, device="cuda")[None, :] < (cu[1:] - cu[:-1])[:, None]
    row = torch.where(held, row, 0)
    q, k, v = (s[n].float().unflatten(-1, (-1, D))[row].transpose(1, 2) for n in "qkv")  # [B][heads][most][D]
    q = q.unflatten(1, (HKV, H // HKV))
    k, v = k[:, :, None], v[:, :, None]
    step = max(1, (1 << 30) // (B * H * most))  # rows of scores that fit in memory at a time
    for a in range(0, most, step):
        z = min(most, a + step)
        score = q[..., a:z, :] @ k[..., :z, :].transpose(-1, -2) * (1.0 / math.sqrt(D))
        i, j = torch.arange(a, z, device="cuda")[:, None], torch.arange(z, device="cuda")[None, :]
        seen = j <= i
        if s["window"]:
            seen &= j > i - s["window"]
        got = (_softmax(score, seen, s["softcap"]) @ v[..., :z, :]).flatten(1, 2).transpose(1, 2).flatten(2)
        s["result"][row[:, a:z][held[:, a:z]]] = got[held[:, a:z]].to(s["result"].dtype)
    return s["result"]


# ------------------------------------------------------------- the entry points

def _plan(s):
    """What a program keeps for its calls: the library, the cache's handle, a workspace, addresses and the stream."""
    from imurun_b200 import native
    s["lib"] = lib = native.load_library()
    s["stream"] = torch.cuda.current_stream().cuda_stream
    if s["op"] == "packed":
        return
    part = lib.fbx_kv4_layer_bytes(s["HKV"], s["D"])
    s["cache"] = native.Kv4Cache(pool=s["pool"].data_ptr(), page_table=s["table"].data_ptr(), err=None,
                                 page_stride=s["layers"] * part, layer_offset=s["layer"] * part,
                                 n_pages=s["pool"].numel() // (s["layers"] * part), table_stride=s["table"].shape[1],
                                 n_seqs=s["table"].shape[0], n_head_kv=s["HKV"], head_dim=s["D"])
    if s["op"] == "decode":
        s["space"] = torch.empty(lib.fbx_kv4_attention_workspace(s["T"], s["H"], s["HKV"], s["D"], s["keys"]),
                                 dtype=torch.uint8, device="cuda")


def _own(s):
    lib, H, HKV, D, t = s["lib"], s["H"], s["HKV"], s["D"], TYPES[s["type"]][0]
    if s["op"] == "append":
        x, w = s["qkv"].data_ptr(), s["qkv"].shape[1]
        size = s["qkv"].element_size()
        rc = lib.fbx_kv4_append(s["cache"], t, x, x + H * D * size, x + (H + HKV) * D * size, w, w, s["T"], H,
                                s["seq"].data_ptr(), s["pos"].data_ptr(), s["rot"], int(s["neox"]), s["cos"].data_ptr(),
                                s["sin"].data_ptr(), s["cos"].shape[0], TYPES[s["out"]][0], s["q_out"].data_ptr(), H * D,
                                s["k_out"].data_ptr(), s["v_out"].data_ptr(), HKV * D, s["stream"])
        out = {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"], "pool": s["pool"]}
    elif s["op"] == "decode":
        rc = lib.fbx_kv4_attention(s["cache"], t, s["q"].data_ptr(), H * D, s["T"], H, s["seq"].data_ptr(),
                                   s["pos"].data_ptr(), s["keys"], 1.0 / math.sqrt(D), s["softcap"], s["window"],
                                   s["result"].data_ptr(), H * D, s["space"].data_ptr(), s["space"].numel(), s["stream"])
        out = s["result"]
    else:
        rc = lib.fbx_attention_packed(t, s["q"].data_ptr(), H * D, s["k"].data_ptr(), s["v"].data_ptr(), HKV * D,
                                      s["q"].shape[0], s["cu"].data_ptr(), len(s["lens"]), H, HKV, D,
                                      1.0 / math.sqrt(D), s["softcap"], s["window"], s["result"].data_ptr(), H * D,
                                      s["stream"])
        out = s["result"]
    if rc:
        raise RuntimeError("%s: %d" % (s["op"], rc))
    return out


def run(state):
    if own:
        return _own(state)
    return {"append": _append, "decode": _decode, "packed": _packed}[state["op"]](state)


# ------------------------------------------------------------ 64 bits, apart

def _attend64(q, k, v, first, softcap, window):
    """One kv head in 64 bits: q [heads][rows][D] at positions first.., k and v [keys][D]."""
    s = torch.einsum("hrd,kd->hrk", q, k) / math.sqrt(q.shape[-1])
    if softcap:
        s = torch.tanh(s / softcap) * softcap
    behind = (first + torch.arange(q.shape[1], device="cuda"))[:, None] - torch.arange(k.shape[0], device="cuda")[None, :]
    off = behind < 0
    if window:
        off |= behind >= window
    s.masked_fill_(off, -math.inf)
    return torch.einsum("hrk,kd->hrd", torch.softmax(s, -1), v)


def _held64(s, pages):
    """What these pages hold in 64 bits, K and V [positions][heads][D], byte by byte as the format says."""
    D, GP, groups = s["D"], _gp(s["D"]), s["D"] // 32
    size = 2 * (8 * D + 64 * GP)
    rec = s["pool"].view(-1, s["layers"], s["HKV"], size)[pages, s["layer"]].transpose(0, 1)  # [heads][pages][bytes]
    out = []
    for base, v in ((0, False), (size // 2, True)):
        at, shift = [], []
        for j in range(PAGE):
            for d in range(D):
                g, m = d // 32, d % 32
                turn = 4 if (j >> 1) & 1 else 0
                at.append(base + j * D // 2 + (2 * groups * ((m // 4) ^ turn) + 2 * g + m % 4 // 2 if v else
                                               4 * groups * (m // 8) + 4 * g + m % 8 // 2))
                shift.append(4 * (d % 2))
        code = (rec[..., torch.tensor(at, device="cuda")] >> torch.tensor(shift, dtype=torch.uint8, device="cuda")) & 15
        scale = rec[..., base + 8 * D:base + 8 * D + 64 * GP].contiguous().view(torch.float16).double()
        d, lo = (x.reshape(*rec.shape[:2], PAGE, GP)[..., :groups].repeat_interleave(32, -1) for x in scale.chunk(2, -1))
        out.append((lo + d * code.reshape(d.shape)).flatten(1, 2).transpose(0, 1))
    return out


def exact(case, seed):
    s = prepare(case, seed)
    H, HKV, D = s["H"], s["HKV"], s["D"]
    G = H // HKV
    if s["op"] == "append":
        x = s["qkv"].double().view(s["T"], H + 2 * HKV, D)
        c, n = s["cos"].double()[s["pos"].long()], s["sin"].double()[s["pos"].long()]
        y, half = x.clone(), s["rot"] // 2
        for i in range(half):
            a, b = (i, i + half) if s["neox"] else (2 * i, 2 * i + 1)
            u, w = x[:, :H + HKV, a], x[:, :H + HKV, b]
            y[:, :H + HKV, a] = u * c[:, i:i + 1] - w * n[:, i:i + 1]
            y[:, :H + HKV, b] = u * n[:, i:i + 1] + w * c[:, i:i + 1]
        out = {"q": y[:, :H].reshape(s["T"], -1), "k": None, "v": None, "pool": None}
        if s["out"] != "f32":
            # a value at the border of two codes goes either way by its last bit in 32: in 16 bits such values are too
            # few to count, against 32 bits they would say nothing
            for name, z in (("k", y[:, H:H + HKV]), ("v", y[:, H + HKV:])):
                z = z.reshape(s["T"], HKV, D // 32, 32)
                low = z.min(-1, keepdim=True).values.to(torch.float32).half().double()
                d = ((z.max(-1, keepdim=True).values - low) / 15).to(torch.float32).half().double()
                code = torch.clamp(torch.round((z - low) / torch.where(d > 0, d, 1.0)), 0, 15)
                out[name] = torch.where(d > 0, low + d * code, low).reshape(s["T"], -1)
        return out
    if s["op"] == "decode":
        out = torch.empty((s["T"], HKV, G, D), dtype=torch.float64, device="cuda")
        for t in range(s["T"]):
            n = int(s["pos"][t]) + 1
            k, v = _held64(s, s["table"][int(s["seq"][t]), :(n + PAGE - 1) // PAGE].long())
            for h in range(HKV):
                q = s["q"][t].double().view(HKV, G, 1, D)[h]
                out[t, h] = _attend64(q, k[:n, h], v[:n, h], n - 1, s["softcap"], s["window"])[:, 0]
        return out.view(s["T"], H * D)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for n in filter(None, s["lens"]):
        q, k, v = (s[x][at:at + n].double().view(n, -1, D) for x in "qkv")
        for h in range(HKV):
            for a in range(0, n, 2048):
                z = min(n, a + 2048)
                got = _attend64(q[a:z, h * G:(h + 1) * G].transpose(0, 1), k[:z, h], v[:z, h], a, s["softcap"], s["window"])
                out[at + a:at + z].view(z - a, H, D)[:, h * G:(h + 1) * G] = got.transpose(0, 1)
        at += n
    return out
