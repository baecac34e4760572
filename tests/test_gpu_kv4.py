"""The paged cache held in 4 bits, attention over it, and attention of packed
prompts (fbx_kv4_append, fbx_kv4_attention, fbx_attention_packed) against
plain forms, on device buffers of torch."""
from __future__ import annotations

import numpy as np
import pytest

import kv4_plain as plain

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from imurun_b200 import native
    return native.load_library(), torch, native


def dtype(torch, t):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[t]


def dev(torch, x, t=None):
    y = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    return y.to(dtype(torch, t)) if t else y


def host(x):
    return x.float().cpu().numpy()


class Cache:
    """A pool with its page tables on the device, and what a record's first byte is."""

    def __init__(self, env, lens, HKV, D, layers=1, layer=0, gap=0, fill=None, seed=0, page_stride=None, spare=2):
        self.lib, self.torch, native = env
        self.HKV, self.D, self.layer = HKV, D, layer
        rng = np.random.default_rng(seed)
        need = [-(-n // plain.PAGE) for n in lens]
        self.n_pages = sum(need) + spare
        order = rng.permutation(self.n_pages).astype(np.int32)
        self.table = np.full((len(lens), max(need + [1]) + 1), -7, np.int32)   # entries past a sequence's end: no page
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        part = HKV * plain.record_bytes(D)
        assert self.lib.fbx_kv4_layer_bytes(HKV, D) == part
        self.stride = page_stride or layers * part + gap
        self.offset = layer * part
        size = self.n_pages * self.stride
        if page_stride:
            self.pool = self.torch.empty(size, dtype=self.torch.uint8, device="cuda")
        else:
            self.pool = dev(self.torch, np.full(size, 0 if fill is None else fill, np.uint8))
        self.dtable = dev(self.torch, self.table)
        self.err = self.torch.zeros(1, dtype=self.torch.int32, device="cuda")
        self.handle = native.Kv4Cache(pool=self.pool.data_ptr(), page_table=self.dtable.data_ptr(),
                                      err=self.err.data_ptr(), page_stride=self.stride, layer_offset=self.offset,
                                      n_pages=self.n_pages, table_stride=self.table.shape[1], n_seqs=len(lens),
                                      n_head_kv=HKV, head_dim=D)

    def record(self, seq, pos, head):
        return int(self.table[seq, pos // plain.PAGE]) * self.stride + self.offset + head * plain.record_bytes(self.D)

    def put(self, pool, seq, pos, k, v):
        """Rows k, v [HKV][D] of one position into the host image `pool`."""
        for head in range(self.HKV):
            for x, is_v in ((k, False), (v, True)):
                plain.store(pool, self.record(seq, pos, head), pos % plain.PAGE, is_v, self.D, *plain.quantise(x[head][None]))

    def random(self, lens, rng, spread=1.0):
        """Fills the sequences with random rows, on host and device; padding rows of the last pages hold what 0xFF means: NaN scales."""
        image = np.full(self.pool.numel(), 0xFF, np.uint8)
        for s, n in enumerate(lens):
            for p in range(n):
                self.put(image, s, p, (rng.standard_normal((self.HKV, self.D)) * spread).astype(np.float32),
                         (rng.standard_normal((self.HKV, self.D)) * spread + 0.3).astype(np.float32))
        self.pool.copy_(dev(self.torch, image))
        return image

    def held(self, image, seq, n, head):
        """K, V and V's d [n][D] in 64 bits of a sequence's first n positions."""
        got = [np.concatenate(x)[:n] for x in zip(*(plain.fetch(image, self.record(seq, i, head), self.D, steps=True)
                                                    for i in range(0, n, plain.PAGE)))]
        return got


def tables(n, rot, base=10000.0):
    f = base ** (-np.arange(0, max(rot, 2), 2) / max(rot, 2))
    a = np.arange(n)[:, None] * f[None, :]
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def call_append(env, c, t, qkv, H, seq, pos, rot, neox, cos, sin, out, told=True, stream=0):
    """fbx_kv4_append on rows q | k | v; returns rc and the outputs (pre-filled with 7)."""
    lib, torch, _ = env
    D, HKV, T = c.D, c.HKV, len(seq)
    q_out, k_out, v_out = (torch.full((T, w * D), 7.0, dtype=dtype(torch, out), device="cuda") for w in (H, HKV, HKV))
    dseq, dpos = dev(torch, np.asarray(seq, np.int32)), dev(torch, np.asarray(pos, np.int32))
    x, es, ld = qkv.data_ptr(), qkv.element_size(), qkv.stride(0)
    rc = lib.fbx_kv4_append(c.handle, plain.TYPE[t], x, x + H * D * es, x + (H + HKV) * D * es, ld, ld, T, H,
                            dseq.data_ptr(), dpos.data_ptr(), rot, int(neox), cos.data_ptr(), sin.data_ptr(),
                            cos.shape[0], plain.TYPE[out], q_out.data_ptr(), H * D, k_out.data_ptr() if told else None,
                            v_out.data_ptr() if told else None, HKV * D, stream)
    torch.cuda.synchronize()
    return rc, q_out, k_out, v_out


APPENDS = [  # type, out, T, lens, H, HKV, D, rot, neox, layers, layer
    ("f32", "f32", 1, [7], 8, 2, 128, 128, False, 1, 0),
    ("f32", "f16", 37, [30, 21], 6, 2, 96, 96, True, 2, 1),
    ("f16", "f16", 50, [20, 17, 40], 5, 5, 64, 64, True, 3, 1),
    ("bf16", "bf16", 33, [50], 14, 2, 128, 64, False, 1, 0),
    ("bf16", "f32", 20, [33, 1], 3, 1, 128, 128, True, 2, 0),
    ("f16", "bf16", 16, [16], 12, 4, 96, 20, False, 1, 0),
    ("f32", "bf16", 9, [9], 2, 2, 64, 22, True, 1, 0),
    ("f16", "f32", 170, [170], 4, 1, 96, 0, False, 1, 0),
    ("bf16", "f16", 5, [90], 8, 8, 64, 2, True, 1, 0),
]


@pytest.mark.parametrize("t,out,T,lens,H,HKV,D,rot,neox,layers,layer", APPENDS)
def test_append_matches_the_format_bit_for_bit(env, t, out, T, lens, H, HKV, D, rot, neox, layers, layer):
    """Cache bytes equal to the plain form's, everything around them untouched;
    stored values and rotated queries rounded once to the output type."""
    lib, torch, _ = env
    rng = np.random.default_rng(T + D + H)
    c = Cache(env, lens, HKV, D, layers, layer, gap=48, fill=0xAB, seed=D)
    where = [(s, p) for s, n in enumerate(lens) for p in range(n)]
    where = [where[i] for i in rng.permutation(len(where))[:T]]   # any order, holes left
    T = len(where)
    seq, pos = [s for s, _ in where], [p for _, p in where]
    # rows in the middle of wider ones, 16 values in front
    wide = dev(torch, plain.round_to(rng.standard_normal((T, (H + 2 * HKV) * D + 32)).astype(np.float32) * 2, t), t)
    qkv = wide[:, 16:16 + (H + 2 * HKV) * D]
    cos, sin = tables(max(lens) + 3, rot)
    rc, q_out, k_out, v_out = call_append(env, c, t, qkv, H, seq, pos, rot, neox, dev(torch, cos), dev(torch, sin), out)
    assert rc == 0 and int(c.err) == 0
    x = host(qkv).reshape(T, H + 2 * HKV, D)
    image = np.full(c.pool.numel(), 0xAB, np.uint8)
    for i, (s, p) in enumerate(where):
        turned = plain.rope(x[i, :H + HKV], cos[p], sin[p], rot, neox)
        c.put(image, s, p, turned[H:], x[i, H + HKV:])
        assert np.array_equal(host(q_out[i]), plain.round_to(turned[:H].reshape(-1), out))
        for got, want in ((k_out, turned[H:]), (v_out, x[i, H + HKV:])):
            assert np.array_equal(host(got[i]), plain.round_to(plain.values(*plain.quantise(want)).reshape(-1), out))
    assert np.array_equal(c.pool.cpu().numpy(), image)


def test_append_stores_what_the_format_says_for_odd_values(env):
    """Constants, zeros, one-sided groups, tiny and huge values, infinities and NaN."""
    lib, torch, _ = env
    D, rows = 64, []
    rng = np.random.default_rng(3)
    for base in (np.zeros(32), np.full(32, 0.1), np.full(32, -3.3), np.arange(32) / 7, np.arange(32) * 1e-7,
                 rng.standard_normal(32) * 1e-9, rng.standard_normal(32) * 3e4, rng.standard_normal(32) * 1e30,
                 np.where(np.arange(32) == 5, np.inf, 1.0), np.where(np.arange(32) == 6, -np.inf, np.arange(32)),
                 np.where(np.arange(32) % 3 == 0, np.nan, np.arange(32) * 0.5), np.full(32, np.nan),
                 np.where(np.arange(32) == 0, 100.0, 1e-3), 1000 + np.arange(32) * 1e-3, np.full(32, 65519.0),
                 np.where(np.arange(32) < 16, np.inf, -np.inf)):
        rows.append(base)
    x = np.concatenate([np.stack(rows), np.stack(rows[::-1])], 1).astype(np.float32)   # two groups a row
    T = len(x)
    c = Cache(env, [T], 1, D, fill=0)
    qkv = dev(torch, np.concatenate([np.zeros((T, D), np.float32), x, x], 1))
    cos, sin = tables(T, 2)
    rc, _, k_out, v_out = call_append(env, c, "f32", qkv, 1, [0] * T, list(range(T)), 0, False, dev(torch, cos),
                                      dev(torch, sin), "f32")
    assert rc == 0
    image = np.zeros(c.pool.numel(), np.uint8)
    for p in range(T):
        c.put(image, 0, p, x[p][None], x[p][None])
    assert np.array_equal(c.pool.cpu().numpy(), image)
    want = plain.values(*plain.quantise(x))
    assert np.array_equal(host(k_out), want) and np.array_equal(host(v_out), want) and np.isfinite(want).all()


def test_append_skips_padding_and_flags_what_is_outside(env):
    lib, torch, _ = env
    H, HKV, D = 4, 2, 128
    c = Cache(env, [20, 20], HKV, D, fill=0x5A)
    cos, sin = tables(64, D)
    qkv = torch.randn((6, (H + 2 * HKV) * D), device="cuda")
    before = c.pool.clone()

    def call(seq, pos):
        c.err.zero_()
        c.pool.copy_(before)
        rc, q, k, v = call_append(env, c, "f32", qkv[:len(seq)], H, seq, pos, D, False, dev(torch, cos), dev(torch, sin), "f32")
        assert rc == 0
        kept = [bool((x[i] == 7).all()) for i in range(len(seq)) for x in (q, k, v)]
        return int(c.err), bool(torch.equal(c.pool, before)), kept

    # padding: nothing written, nothing flagged
    assert call([0, 5, -1], [-1, -1, -9]) == (0, True, [True] * 9)
    # a sequence outside the tables, a position past the rotation's or the page table
    assert call([2, -1, 0], [0, 0, 64]) == (6, True, [True] * 9)
    assert call([0], [63]) == (6, True, [True] * 3)
    # a table entry that names no page
    assert call([0, 1], [47, 40]) == (5, True, [True] * 6)
    # good tokens beside bad ones are stored
    flag, same, kept = call([0, 9, 1], [3, 0, 19])
    assert flag == 6 and not same and kept == [False] * 3 + [True] * 3 + [False] * 3


def test_append_in_place_and_without_outputs(env):
    """Rotating q in its own rows, K and V replaced by what the cache holds; no
    outputs at all: the same cache."""
    lib, torch, _ = env
    for D, rot in ((128, 128), (96, 96), (64, 32)):
        H, HKV, T = 7, 2, 21
        cos, sin = (dev(torch, x) for x in tables(T, rot))
        seq, pos = dev(torch, np.zeros(T, np.int32)), dev(torch, np.arange(T, dtype=np.int32))
        qkv = torch.randn((T, (H + 2 * HKV) * D), device="cuda").to(torch.bfloat16)
        a, b, e = (Cache(env, [T], HKV, D, seed=1) for _ in range(3))
        rc, q_out, k_out, v_out = call_append(env, a, "bf16", qkv, H, [0] * T, list(range(T)), rot, True, cos, sin, "bf16")
        assert rc == 0
        x, ld = qkv.clone(), qkv.shape[1]
        p = [x.data_ptr() + 2 * D * o for o in (0, H, H + HKV)]
        assert lib.fbx_kv4_append(b.handle, 30, *p, ld, ld, T, H, seq.data_ptr(), pos.data_ptr(), rot, 1, cos.data_ptr(),
                                  sin.data_ptr(), T, 30, p[0], ld, p[1], p[2], ld, None) == 0
        y = qkv.clone()
        p = [y.data_ptr() + 2 * D * o for o in (0, H, H + HKV)]
        assert lib.fbx_kv4_append(e.handle, 30, None, p[1], p[2], 0, ld, T, 0, seq.data_ptr(), pos.data_ptr(), rot, 1,
                                  cos.data_ptr(), sin.data_ptr(), T, 30, None, 0, None, None, 0, None) == 0
        torch.cuda.synchronize()
        assert torch.equal(x, torch.cat((q_out, k_out, v_out), 1)) and torch.equal(y, qkv)
        assert torch.equal(a.pool, b.pool) and torch.equal(a.pool, e.pool)


def attention(env, c, t, q, H, seq, pos, max_keys, scale, softcap=0.0, window=0, stream=None, fill=7.0):
    lib, torch, _ = env
    T = len(seq)
    out = torch.full((T, H * c.D), fill, dtype=dtype(torch, t), device="cuda")
    dseq, dpos = dev(torch, np.asarray(seq, np.int32)), dev(torch, np.asarray(pos, np.int32))
    size = lib.fbx_kv4_attention_workspace(T, H, c.HKV, c.D, max_keys)
    ws = torch.full((max(size, 16),), 0xFF, dtype=torch.uint8, device="cuda")
    rc = lib.fbx_kv4_attention(c.handle, plain.TYPE[t], q.data_ptr(), q.stride(0), T, H, dseq.data_ptr(), dpos.data_ptr(),
                               max_keys, scale, softcap, window, out.data_ptr(), H * c.D, ws.data_ptr(), size, stream)
    torch.cuda.synchronize()
    assert rc == 0
    return out


def near(got, want, size, t, softcap=0.0):
    """size: what plain.attend() says with steps. A weight times its group's d is rounded to f16 for 16-bit types, to two
    f16 parts for f32."""
    mean, ext, coarse = size
    tol = plain.allowed(want, mean, ext, t, 2.0 ** -22 if t == "f32" else 2.0 ** -11, softcap, coarse)
    off = np.abs(got - want)
    assert (off <= tol).all(), (off / tol).max()


ATTENTIONS = [  # type, H, HKV, D, positions, softcap, window
    ("f32", 8, 2, 128, [0, 1, 14, 15, 16, 17, 31, 32, 100], 0.0, 0),
    ("f16", 8, 8, 64, [0, 63, 64, 200, 257], 0.0, 0),
    ("bf16", 14, 2, 128, [300, 5, 0], 0.0, 0),
    ("f32", 12, 4, 96, [77, 33, 15], 0.0, 0),
    ("bf16", 9, 1, 96, [129, 0, 48], 30.0, 0),
    ("f32", 24, 2, 64, [260, 19], 5.0, 50),
    ("f16", 16, 2, 128, [500, 40, 16, 15], 0.0, 17),
    ("f32", 5, 1, 128, [400, 3], 0.0, 1),
    ("bf16", 4, 4, 64, [90, 31], 0.0, 1000),
]


@pytest.mark.parametrize("t,H,HKV,D,pos,softcap,window", ATTENTIONS)
def test_attention_over_the_cache(env, t, H, HKV, D, pos, softcap, window):
    """Against 64 bits; stale rows of the last page hold NaN scales, page-table entries past the end no page."""
    lib, torch, _ = env
    rng = np.random.default_rng(H + D + len(pos))
    lens = [p + 1 for p in pos]
    c = Cache(env, lens, HKV, D, layers=2, layer=1, gap=16, seed=2)
    image = c.random(lens, rng)
    T, G = len(pos), H // HKV
    order = rng.permutation(T)
    seq, at = [int(i) for i in order], [pos[i] for i in order]
    q = dev(torch, plain.round_to(rng.standard_normal((T, H * D + 8)).astype(np.float32) * 1.5, t), t)[:, 8:] \
        if t != "f32" else dev(torch, rng.standard_normal((T, H * D + 8)).astype(np.float32) * 1.5)[:, 8:]
    scale = 1.0 / np.sqrt(D)
    for most in (max(lens), 1, 100000):   # any bound gives the right result
        out = host(attention(env, c, t, q, H, seq, at, most, scale, softcap, window))
        assert int(c.err) == 0
        x = host(q).reshape(T, H, D)
        for i in range(T):
            for hk in range(HKV):
                k, v, d = c.held(image, seq[i], at[i] + 1, hk)
                want, *size = plain.attend(x[i, hk * G:(hk + 1) * G], k, v, [at[i]] * G, scale, softcap, window, d)
                near(out[i].reshape(H, D)[hk * G:(hk + 1) * G], want, size, t, softcap)


@pytest.mark.parametrize("t,spread,size", [("f32", 1e-4, 1e4), ("f16", 1e-4, 1e3), ("bf16", 1e-6, 1e6), ("f32", 300.0, 1e-3),
                                            ("bf16", 3000.0, 1e-5), ("f32", 1.0, 0.0)])
def test_attention_of_tiny_and_huge_values(env, t, spread, size):
    """Cache values and queries far from 1: no part of the sum may leave the range of 16 bits."""
    lib, torch, _ = env
    rng = np.random.default_rng(9)
    H, HKV, D, pos = 4, 1, 128, [250]
    c = Cache(env, [251], HKV, D)
    image = c.random([251], rng, spread)
    q = dev(torch, plain.round_to((rng.standard_normal((1, H * D)) * size).astype(np.float32), t), t)
    out = host(attention(env, c, t, q, H, [0], pos, 251, 1.0 / np.sqrt(D))).reshape(H, D)
    k, v, d = c.held(image, 0, 251, 0)
    want, *size = plain.attend(host(q).reshape(H, D), k, v, pos * H, 1.0 / np.sqrt(D), steps=d)
    # f16 outputs below its normal range: half of its smallest step, 2^-25, in allowed()
    near(out, want, size, t)


def test_attention_padding_and_bad_pages(env):
    lib, torch, _ = env
    H, HKV, D = 8, 2, 128
    rng = np.random.default_rng(4)
    c = Cache(env, [40, 40], HKV, D)
    image = c.random([40, 40], rng)
    q = torch.randn((3, H * D), device="cuda")
    # padding rows stay, whatever their sequence
    out = attention(env, c, "f32", q, H, [0, -3, 1], [-1, -1, 39], 40, 0.1)
    assert int(c.err) == 0 and bool((out[:2] == 7).all()) and bool((out[2] != 7).any())
    # an unknown sequence: flagged, nothing seen, zeros
    out = attention(env, c, "f32", q, H, [2, 1, 0], [5, 39, 39], 40, 0.1)
    assert int(c.err) == 6 and bool((out[0] == 0).all()) and bool(torch.isfinite(out).all())
    c.err.zero_()
    # a page that is not in the pool, in the middle: its keys are not seen
    c.dtable[0, 1] = c.n_pages
    out = host(attention(env, c, "f32", q[:1], H, [0], [39], 40, 0.1)).reshape(H, D)
    assert int(c.err) == 5
    keep = np.r_[0:16, 32:40]
    for hk in range(HKV):
        k, v, d = c.held(image, 0, 40, hk)
        want, *size = plain.attend(host(q)[0].reshape(H, D)[hk * 4:hk * 4 + 4], k[keep], v[keep], [23] * 4, 0.1, steps=d[keep])
        near(out[hk * 4:hk * 4 + 4], want, size, "f32")
    # a position past the page table is flagged; the keys 40..47 that it does see hold NaN, as the formula has it
    c.err.zero_()
    out = attention(env, c, "f32", q[:1], H, [1], [1000], 1001, 0.1)
    assert int(c.err) in (5, 6) and bool(torch.isnan(out).all())


def test_cache_past_four_gigabytes(env):
    """Pages 1.5 GiB apart: byte offsets past 32 bits in the append and in the attention."""
    lib, torch, _ = env
    H, HKV, D, n = 4, 2, 128, 60
    c = Cache(env, [n], HKV, D, page_stride=3 << 29, spare=0)
    rng = np.random.default_rng(5)
    x = torch.from_numpy(rng.standard_normal((n, (H + 2 * HKV) * D)).astype(np.float32)).cuda()
    cos, sin = (dev(torch, a) for a in tables(n, D))
    rc, q, k, v = call_append(env, c, "f32", x, H, [0] * n, list(range(n)), D, True, cos, sin, "f32")
    assert rc == 0 and int(c.err) == 0
    out = host(attention(env, c, "f32", q[-1:], H, [0], [n - 1], n, 0.08)).reshape(H, D)
    kk, vv = (host(y).reshape(n, HKV, D) for y in (k, v))
    d = plain.quantise(host(x)[:, (H + HKV) * D:].reshape(n, HKV, D))[1].astype(np.float64).repeat(32, -1)
    for hk in range(HKV):
        want, *size = plain.attend(host(q)[-1].reshape(H, D)[hk * 2:hk * 2 + 2], kk[:, hk], vv[:, hk], [n - 1] * 2, 0.08,
                                   steps=d[:, hk])
        near(out[hk * 2:hk * 2 + 2], want, size, "f32")


# ------------------------------------------------------------------ packed prompts

def packed(env, t, q, k, v, cu, H, HKV, D, scale, softcap=0.0, window=0, out=None, stream=None, rows=None):
    lib, torch, _ = env
    if out is None:
        out = torch.full((q.shape[0], H * D), 7.0, dtype=q.dtype, device="cuda")
    rc = lib.fbx_attention_packed(plain.TYPE[t], q.data_ptr(), q.stride(0), k.data_ptr(), v.data_ptr(), k.stride(0),
                                  q.shape[0] if rows is None else rows, cu.data_ptr(), cu.numel() - 1, H, HKV, D, scale,
                                  softcap, window, out.data_ptr(), out.stride(0), stream)
    assert rc == 0
    torch.cuda.synchronize()
    return out


PACKED = [  # type, lens, H, HKV, D, softcap, window
    ("bf16", [1], 4, 2, 128, 0.0, 0),
    ("f16", [0, 1, 0, 2, 17, 0], 3, 1, 64, 0.0, 0),
    ("bf16", [127, 128, 129], 2, 2, 128, 0.0, 0),
    ("f16", [255, 256, 257], 4, 1, 128, 0.0, 0),
    ("f16", [300, 40, 131], 6, 2, 96, 0.0, 0),
    ("bf16", [64, 65, 63, 1, 513], 2, 1, 64, 0.0, 0),
    ("bf16", [385, 5], 8, 1, 128, 20.0, 0),
    ("f16", [400, 33], 4, 4, 64, 0.0, 1),
    ("f16", [390, 200], 2, 1, 128, 0.0, 100),
    ("bf16", [520, 128], 4, 2, 96, 8.0, 128),
    ("bf16", [600], 2, 2, 64, 0.0, 257),
]


def packed_reference(q, k, v, lens, H, HKV, D, scale, softcap, window):
    G, at = H // HKV, 0
    want, bound = np.zeros(q.shape), np.zeros(q.shape)
    mean, ext = np.zeros(q.shape), np.zeros((len(q), H))
    for n in lens:
        for h in range(H):
            a, b = slice(h * D, h * D + D), slice(h // G * D, h // G * D + D)
            want[at:at + n, a], mean[at:at + n, a], ext[at:at + n, h] = plain.attend(
                q[at:at + n, a], k[at:at + n, b], v[at:at + n, b], range(n), scale, softcap, window)
        at += n
    return want, mean, ext


def check_packed(got, want, mean, ext, H, D, t, softcap, rows):
    for h in range(H):
        a = slice(h * D, h * D + D)
        # a weight is rounded to the type before its product with v
        tol = plain.allowed(want[:rows, a], mean[:rows, a], ext[:rows, h], t, plain.HALF[t], softcap)
        off = np.abs(got[:rows, a] - want[:rows, a])
        assert (off <= tol).all(), (h, (off / tol).max())


@pytest.mark.parametrize("t,lens,H,HKV,D,softcap,window", PACKED)
def test_packed_prompts(env, t, lens, H, HKV, D, softcap, window):
    """Rows inside wider ones; rows after the last sequence hold NaN and keep what out had."""
    lib, torch, _ = env
    rng = np.random.default_rng(sum(lens) + D + H)
    N, extra = sum(lens), 5
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    wide = rng.standard_normal((N + extra, (H + 2 * HKV) * D + 8)).astype(np.float32)
    wide[N:] = np.nan
    wide = dev(torch, wide, t)
    q, k, v = wide[:, 8:8 + H * D], wide[:, 8 + H * D:8 + (H + HKV) * D], wide[:, 8 + (H + HKV) * D:]
    scale = 1.7 / np.sqrt(D)
    out = packed(env, t, q, k, v, dev(torch, cu), H, HKV, D, scale, softcap, window)
    assert bool((out[N:] == 7).all())
    ref = packed_reference(host(q)[:N], host(k)[:N], host(v)[:N], lens, H, HKV, D, scale, softcap, window)
    check_packed(host(out), *ref, H, D, t, softcap, N)


@pytest.mark.parametrize("t,D", [("f16", 64), ("bf16", 128), ("f16", 96)])
def test_packed_masked_infinities_and_nan(env, t, D):
    """A row's output does not depend on what later rows, or other sequences,
    hold, even where that is not finite; rows that see it follow the formula."""
    lib, torch, _ = env
    rng = np.random.default_rng(D)
    lens, H, HKV = [150, 90, 300], 4, 2
    N = sum(lens)
    cu = dev(torch, np.concatenate([[0], np.cumsum(lens)]).astype(np.int32))
    q, k, v = (dev(torch, rng.standard_normal((N, h * D)).astype(np.float32), t) for h in (H, HKV, HKV))
    scale = 1.0 / np.sqrt(D)
    clean = packed(env, t, q, k, v, cu, H, HKV, D, scale)
    for row, what in ((149, np.nan), (100, np.inf), (239, -np.inf), (240 + 17, np.nan), (240 + 200, np.inf)):
        seq_end = next(e for e in np.cumsum(lens) if row < e)
        vv, kk = v.clone(), k.clone()
        vv[row, D + 3] = what          # kv head 1, dimension 3
        out = packed(env, t, q, k, vv, cu, H, HKV, D, scale)
        hit = torch.zeros_like(out, dtype=torch.bool)
        for h in (2, 3):
            hit[row:seq_end, h * D + 3] = True
        assert torch.equal(out[~hit], clean[~hit]), (row, what)
        want = torch.full_like(out, what)
        assert torch.equal(torch.isnan(out[hit]), torch.isnan(want[hit])) and torch.equal(
            out[hit][~torch.isnan(want[hit])], want[hit][~torch.isnan(want[hit])])
        kk[row, 5] = np.nan            # a key of head 0: every row from it on loses heads 0 and 1
        out = packed(env, t, q, kk, v, cu, H, HKV, D, scale)
        hit = torch.zeros_like(out, dtype=torch.bool)
        hit[row:seq_end, :2 * D] = True
        assert torch.equal(out[~hit], clean[~hit]) and bool(torch.isnan(out[hit]).all())
    # under a window, rows behind it stop seeing the row
    vv = v.clone()
    vv[160, 7] = np.inf
    a = packed(env, t, q, k, v, cu, H, HKV, D, scale, window=20)
    b = packed(env, t, q, k, vv, cu, H, HKV, D, scale, window=20)
    hit = torch.zeros_like(a, dtype=torch.bool)
    for h in (0, 1):
        hit[160:180, h * D + 7] = True
    assert torch.equal(a[~hit], b[~hit]) and bool(torch.isinf(b[hit]).all())


def test_packed_large_scores_and_bad_lengths(env):
    lib, torch, _ = env
    H, HKV, D, N = 2, 1, 128, 300
    q = torch.randn((N, H * D), device="cuda").bfloat16() * 60
    k, v = (torch.randn((N, HKV * D), device="cuda").bfloat16() for _ in range(2))
    cu = dev(torch, np.array([0, N], np.int32))
    out = host(packed(env, "bf16", q, k, v, cu, H, HKV, D, 1.0))       # scores of several hundred
    ref = packed_reference(host(q), host(k), host(v), [N], H, HKV, D, 1.0, 0.0, 0)
    check_packed(out, *ref, H, D, "bf16", 0.0, N)
    # ends past the rows and ends before starts: read and written inside the buffers only
    cu = dev(torch, np.array([0, 100, 90, 5000, 20], np.int32))
    out = packed(env, "bf16", q, k, v, cu, H, HKV, D, 0.1)
    assert bool(torch.isfinite(out).all())


# ---------------------------------------------------- as they are used, together

@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_prompts_then_tokens(env, t):
    """Prompts of a batch are appended and attended, then tokens one by one:
    every output against 64 bits over the values that the cache holds."""
    lib, torch, _ = env
    rng = np.random.default_rng(11)
    H, HKV, D, rot, lens, steps = 8, 2, 128, 128, [45, 3, 130], 20
    G, scale, B = H // HKV, 1.0 / np.sqrt(D), len(lens)
    c = Cache(env, [n + steps for n in lens], HKV, D)
    cos, sin = (dev(torch, x) for x in tables(200, rot))
    seq = [s for s, n in enumerate(lens) for _ in range(n)]
    pos = [p for n in lens for p in range(n)]
    qkv = dev(torch, rng.standard_normal((len(seq), (H + 2 * HKV) * D)).astype(np.float32), t)
    rc, q, k, v = call_append(env, c, t, qkv, H, seq, pos, rot, True, cos, sin, t)
    assert rc == 0
    cu = dev(torch, np.concatenate([[0], np.cumsum(lens)]).astype(np.int32))
    out = host(packed(env, t, q, k, v, cu, H, HKV, D, scale))
    check_packed(out, *packed_reference(host(q), host(k), host(v), lens, H, HKV, D, scale, 0.0, 0), H, D, t, 0.0, len(seq))
    for step in range(steps):
        at = [n + step for n in lens]
        qkv = dev(torch, rng.standard_normal((B, (H + 2 * HKV) * D)).astype(np.float32), t)
        rc, q, _, _ = call_append(env, c, t, qkv, H, list(range(B)), at, rot, True, cos, sin, t)
        assert rc == 0
        if step % 5 and step != steps - 1:
            continue
        got = host(attention(env, c, t, q, H, list(range(B)), at, max(at) + 1, scale)).reshape(B, H, D)
        image = c.pool.cpu().numpy()
        for s in range(B):
            for hk in range(HKV):
                kk, vv, d = c.held(image, s, at[s] + 1, hk)
                hs = slice(hk * G, hk * G + G)
                want, *size = plain.attend(host(q)[s].reshape(H, D)[hs], kk, vv, [at[s]] * G, scale, steps=d)
                near(got[s, hs], want, size, t)
    assert int(c.err) == 0


def test_captured_and_replayed_on_a_side_stream(env):
    """append -> attention, and packed attention, captured once on a side
    stream and replayed on new inputs in the same buffers; two graphs with
    workspaces of their own, replayed at the same time, give what eager calls give."""
    lib, torch, _ = env
    H, HKV, D, T, n = 8, 2, 128, 3, 400
    rng = np.random.default_rng(12)
    cos, sin = (dev(torch, x) for x in tables(n + 8, D))
    graphs = []
    for g in range(2):
        c = Cache(env, [n + 8] * T, HKV, D, seed=g)
        c.random([n] * T, rng)
        b = {"c": c, "qkv": torch.randn((T, (H + 2 * HKV) * D), device="cuda").half(),
             "seq": torch.arange(T, dtype=torch.int32, device="cuda"),
             "pos": torch.full((T,), n, dtype=torch.int32, device="cuda"),
             "q": torch.zeros((T, H * D), dtype=torch.float16, device="cuda"),
             "out": torch.zeros((T, H * D), dtype=torch.float16, device="cuda"),
             "cu": dev(torch, np.array([0, 1, T], np.int32)),
             "ws": torch.zeros(max(16, lib.fbx_kv4_attention_workspace(T, H, HKV, D, n + 8)), dtype=torch.uint8, device="cuda")}
        b["pk"] = torch.zeros_like(b["out"])

        def calls(b=b, c=c, st=None):
            x = b["qkv"].data_ptr()
            ld = b["qkv"].shape[1]
            p = (x, x + 2 * H * D, x + 2 * (H + HKV) * D)
            assert lib.fbx_kv4_append(c.handle, 1, *p, ld, ld, T, H, b["seq"].data_ptr(), b["pos"].data_ptr(), D, 0,
                                      cos.data_ptr(), sin.data_ptr(), n + 8, 1, b["q"].data_ptr(), H * D, None, None, 0, st) == 0
            assert lib.fbx_kv4_attention(c.handle, 1, b["q"].data_ptr(), H * D, T, H, b["seq"].data_ptr(),
                                         b["pos"].data_ptr(), n + 8, 0.09, 0.0, 0, b["out"].data_ptr(), H * D,
                                         b["ws"].data_ptr(), b["ws"].numel(), st) == 0
            assert lib.fbx_attention_packed(1, *(p[0], ld, p[1], p[2], ld), T, b["cu"].data_ptr(), 2, H, HKV, D, 0.09,
                                            0.0, 0, b["pk"].data_ptr(), H * D, st) == 0

        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            calls(st=torch.cuda.current_stream().cuda_stream)   # the very first call of these shapes may be captured
        graphs.append((graph, stream, b, calls))
    torch.cuda.synchronize()
    for step in range(4):
        for graph, stream, b, _ in graphs:
            b["qkv"].copy_(torch.randn(b["qkv"].shape, device="cuda"))
            b["pos"].fill_(n + step)
            b["out"].fill_(7)
        torch.cuda.synchronize()
        for graph, stream, b, _ in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for graph, stream, b, calls in graphs:
            got, pk, pool = b["out"].clone(), b["pk"].clone(), b["c"].pool.clone()
            b["out"].fill_(3)
            b["pk"].fill_(3)
            calls()
            torch.cuda.synchronize()
            assert torch.equal(got, b["out"]) and torch.equal(pk, b["pk"]) and torch.equal(pool, b["c"].pool)
            assert int(b["c"].err) == 0


def test_calls_allocate_nothing_and_refuse_foreign_memory(env):
    lib, torch, _ = env
    H, HKV, D, n = 8, 2, 128, 64
    c = Cache(env, [n], HKV, D)
    q = torch.randn((1, H * D), device="cuda")
    host_q = np.zeros((1, H * D + 8), np.float32)
    addr = (host_q.ctypes.data + 15) // 16 * 16
    seq = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.zeros_like(q)
    ws = torch.zeros(max(16, lib.fbx_kv4_attention_workspace(1, H, HKV, D, n)), dtype=torch.uint8, device="cuda")

    def call(qp):
        return lib.fbx_kv4_attention(c.handle, 0, qp, H * D, 1, H, seq.data_ptr(), seq.data_ptr(), n, 0.1, 0.0, 0,
                                     out.data_ptr(), H * D, ws.data_ptr(), ws.numel(), None)

    assert call(q.data_ptr()) == 0
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    for _ in range(20):
        assert call(q.data_ptr()) == 0
    torch.cuda.synchronize()
    assert torch.cuda.mem_get_info()[0] == free
    assert call(addr) == -1   # a host array
    torch.cuda.synchronize()


# ------------------------------------------------------------------ larger calls

def filled(env, lens, HKV, D, seed, spread=1.0):
    """A cache filled by fbx_kv4_append without rotation, and the values that it holds, K, V and V's d [rows][HKV][D] f64."""
    lib, torch, _ = env
    c = Cache(env, lens, HKV, D, seed=seed)
    torch.manual_seed(seed)
    seq = np.concatenate([np.full(n, s) for s, n in enumerate(lens)])
    pos = np.concatenate([np.arange(n) for n in lens])
    x = torch.randn((len(seq), 2 * HKV * D), device="cuda") * spread
    x[:, HKV * D:] += 0.25
    cos, sin = (dev(torch, a) for a in tables(max(lens), 2))
    k, v = (torch.empty((len(seq), HKV * D), device="cuda") for _ in range(2))
    dseq, dpos = dev(torch, seq.astype(np.int32)), dev(torch, pos.astype(np.int32))
    ld = x.shape[1]
    assert lib.fbx_kv4_append(c.handle, 0, None, x.data_ptr(), x.data_ptr() + 4 * HKV * D, 0, ld, len(seq), 0, dseq.data_ptr(),
                              dpos.data_ptr(), 0, 0, cos.data_ptr(), sin.data_ptr(), max(lens), 0, None, 0, k.data_ptr(),
                              v.data_ptr(), HKV * D, None) == 0
    torch.cuda.synchronize()
    y = x[:, HKV * D:].view(-1, HKV, D // 32, 32)
    d = ((y.amax(-1) - y.amin(-1)) / 15 + 1e-3).double().repeat_interleave(32, -1)   # no less than the d that is stored
    return c, k.view(-1, HKV, D).double(), v.view(-1, HKV, D).double(), d, np.concatenate([[0], np.cumsum(lens)])


@pytest.mark.parametrize("t,H,HKV,D,lens,window", [
    ("bf16", 8, 1, 128, [6001, 2900, 17], 0),          # more than eight splits: a second launch joins them
    ("f32", 24, 2, 64, [1000] * 19 + [3], 0),          # heads in two runs of eight, clusters
    ("f16", 4, 4, 96, [700, 260, 130, 513], 0),
    ("f16", 16, 8, 128, [300, 40, 2000, 5], 64),
    ("f32", 9, 1, 128, [4000], 2500),
    ("bf16", 6, 2, 128, list(range(1, 180)), 0),       # many tokens, one CTA each
])
def test_attention_over_long_caches(env, t, H, HKV, D, lens, window):
    lib, torch, _ = env
    c, k, v, d, at = filled(env, lens, HKV, D, seed=H + D)
    T, G, scale = len(lens), H // HKV, 1.3 / np.sqrt(D)
    torch.manual_seed(1)
    q = torch.randn((T, H * D), device="cuda").to(dtype(torch, t))
    out = attention(env, c, t, q, H, list(range(T)), [n - 1 for n in lens], max(lens), scale, 0.0, window)
    assert int(c.err) == 0
    for s, n in enumerate(lens):
        a = max(0, n - window) if window else 0
        rows = slice(at[s] + a, at[s] + n)
        x = q[s].view(HKV, G, D).double()
        kk, vv, dd = (y[rows].transpose(0, 1) for y in (k, v, d))
        w = torch.softmax(x @ kk.transpose(1, 2) * scale, -1)
        want, mean, coarse = (z.reshape(H, D).cpu().numpy() for z in (w @ vv, w @ vv.abs(), w @ dd))
        ext = (x.abs() @ kk.abs().transpose(1, 2)).amax(-1).reshape(H).cpu().numpy() * scale
        near(host(out[s]).reshape(H, D), want, (mean, ext, coarse), t)


def test_attention_tokens_of_one_sequence(env):
    """Several tokens of a sequence in one call, as a draft's verification has them: each sees its own past, and each row
    has the bits that it has alone with the same bound."""
    lib, torch, _ = env
    H, HKV, D, n = 8, 2, 128, 333
    c, k, v, d, _ = filled(env, [n], HKV, D, seed=3)
    q = torch.randn((6, H * D), device="cuda")
    pos = [n - 1, 100, n - 1, 0, 15, 16]
    out = attention(env, c, "f32", q, H, [0] * 6, pos, n, 0.1)
    for i, p in enumerate(pos):
        x = q[i].view(HKV, 4, D).double()
        kk, vv, dd = (y[:p + 1].transpose(0, 1) for y in (k, v, d))
        w = torch.softmax(x @ kk.transpose(1, 2) * 0.1, -1)
        want, mean, coarse = (z.reshape(H, D).cpu().numpy() for z in (w @ vv, w @ vv.abs(), w @ dd))
        ext = (x.abs() @ kk.abs().transpose(1, 2)).amax(-1).reshape(H).cpu().numpy() * 0.1
        near(host(out[i]).reshape(H, D), want, (mean, ext, coarse), "f32")
    again = attention(env, c, "f32", q, H, [0] * 6, pos, n, 0.1)
    assert torch.equal(out, again)


def test_attention_keeps_nan_queries(env):
    """A NaN or infinite query gives NaN in its own head and nowhere else."""
    lib, torch, _ = env
    H, HKV, D = 8, 2, 64
    c, *_ = filled(env, [200], HKV, D, seed=4)
    for t in ("f32", "f16", "bf16"):
        q = torch.randn((1, H * D), device="cuda").to(dtype(torch, t))
        clean = attention(env, c, t, q, H, [0], [199], 200, 0.1)
        q[0, 2 * D + 5], q[0, 7 * D] = float("nan"), float("inf")
        out = attention(env, c, t, q, H, [0], [199], 200, 0.1).view(H, D)
        assert bool(torch.isnan(out[2]).all()) and bool(torch.isnan(out[7]).all())
        keep = [0, 1, 3, 4, 5, 6]
        assert torch.equal(out[keep], clean.view(H, D)[keep])


def packed64(torch, q, k, v, lens, H, HKV, D, scale, softcap, window):
    """packed_reference on the device, for longer sequences."""
    G, at = H // HKV, 0
    want, mean = (torch.zeros(q.shape, dtype=torch.float64, device="cuda") for _ in range(2))
    ext = torch.zeros((len(q), H), dtype=torch.float64, device="cuda")
    for n in lens:
        if not n:
            continue
        x, kk, vv = (y[at:at + n].double().view(n, -1, D).transpose(0, 1) for y in (q, k, v))
        kk, vv = kk.repeat_interleave(G, 0), vv.repeat_interleave(G, 0)
        s = x @ kk.transpose(1, 2) * scale
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        i = torch.arange(n, device="cuda")
        off = i[None, :] > i[:, None]
        if window:
            off |= i[None, :] <= i[:, None] - window
        w = torch.softmax(s.masked_fill(off, -float("inf")), -1)
        want[at:at + n] = (w @ vv).transpose(0, 1).reshape(n, -1)
        mean[at:at + n] = (w @ vv.abs()).transpose(0, 1).reshape(n, -1)
        ext[at:at + n] = ((x.abs() @ kk.abs().transpose(1, 2)).masked_fill(off, 0).amax(-1) * scale).T
        at += n
    return want.cpu().numpy(), mean.cpu().numpy(), ext.cpu().numpy()


def many(seed, count, low, high):
    r = np.random.default_rng(seed)
    return [int(n) for n in r.integers(low, high, count)]


@pytest.mark.parametrize("t,lens,H,HKV,D,softcap,window", [
    ("bf16", many(1, 40, 0, 700), 16, 4, 128, 0.0, 0),       # several jobs a CTA
    ("f16", many(2, 100, 0, 90), 5, 1, 64, 0.0, 0),          # more sequences than a warp has lanes
    ("f16", [0] * 50 + [333] + [0] * 40 + [1, 129], 28, 4, 96, 0.0, 0),
    ("bf16", [150, 3], 128, 1, 64, 0.0, 0),                  # the widest group: a row a tile
    ("f16", [40, 130], 50, 1, 128, 0.0, 0),
    ("bf16", [5000], 2, 1, 128, 0.0, 300),
    ("f16", many(3, 9, 100, 1500), 6, 2, 64, 15.0, 500),
    ("bf16", [3001, 17], 7, 1, 128, 0.0, 0),
    ("bf16", many(4, 1000, 0, 60), 4, 2, 64, 0.0, 0),         # so many sequences that they are taken one by one
    ("f16", [0] * 700 + [400] + many(5, 300, 0, 4) + [0] * 100, 3, 1, 128, 0.0, 0),
])
def test_packed_many_jobs(env, t, lens, H, HKV, D, softcap, window):
    lib, torch, _ = env
    torch.manual_seed(sum(lens))
    N = sum(lens)
    q, k, v = (torch.randn((N, h * D), device="cuda").to(dtype(torch, t)) for h in (H, HKV, HKV))
    cu = dev(torch, np.concatenate([[0], np.cumsum(lens)]).astype(np.int32))
    scale = 1.5 / np.sqrt(D)
    out = packed(env, t, q, k, v, cu, H, HKV, D, scale, softcap, window)
    check_packed(host(out), *packed64(torch, q, k, v, lens, H, HKV, D, scale, softcap, window), H, D, t, softcap, N)
    assert torch.equal(out, packed(env, t, q, k, v, cu, H, HKV, D, scale, softcap, window))


def test_packed_rising_scores(env):
    """Scores that grow by far more than the reference's slack from tile to tile: the accumulator is rescaled all the way."""
    lib, torch, _ = env
    H, HKV, D, N = 4, 2, 128, 1400
    torch.manual_seed(5)
    q = torch.ones((N, H * D), device="cuda").bfloat16()
    k = (torch.randn((N, HKV * D), device="cuda") * 0.05 + torch.arange(N, device="cuda")[:, None] * 0.01).bfloat16()
    v = torch.randn((N, HKV * D), device="cuda").bfloat16()
    cu = dev(torch, np.array([0, N], np.int32))
    for scale in (0.05, 1.0):
        out = packed(env, "bf16", q, k, v, cu, H, HKV, D, scale)
        check_packed(host(out), *packed64(torch, q, k, v, [N], H, HKV, D, scale, 0.0, 0), H, D, "bf16", 0.0, N)


def test_packed_rows_past_32_bits(env):
    """Rows so wide that their byte offsets pass 32 bits."""
    lib, torch, _ = env
    H, HKV, D, N, ld = 2, 1, 128, 300, 1 << 23   # 16 MiB a row
    torch.manual_seed(6)
    wide = torch.empty((N, ld), dtype=torch.float16, device="cuda")
    wide[:, :4 * D] = torch.randn((N, 4 * D), device="cuda").half()
    q, k, v = wide[:, :H * D], wide[:, H * D:3 * D], wide[:, 3 * D:4 * D]
    out = torch.empty((N, ld), dtype=torch.float16, device="cuda")[:, :H * D]
    cu = dev(torch, np.array([0, 170, N], np.int32))
    packed(env, "f16", q, k, v, cu, H, HKV, D, 0.1, out=out)
    check_packed(host(out), *packed64(torch, q, k, v, [170, 130], H, HKV, D, 0.1, 0.0, 0), H, D, "f16", 0.0, N)


def test_attention_of_huge_queries(env):
    """f32 queries near the top of their range: scores are finite, and so is the result."""
    lib, torch, _ = env
    H, HKV, D = 2, 1, 64
    c, *_ = filled(env, [40], HKV, D, seed=9)
    q = torch.randn((1, H * D), device="cuda")
    base = attention(env, c, "f32", q, H, [0], [39], 40, 2.0**-3)
    out = attention(env, c, "f32", q * 2.0**118, H, [0], [39], 40, 2.0**-121)
    assert torch.equal(out, base)   # powers of two only


@pytest.mark.parametrize("cap", [1e3, 1e6, 1e12])
def test_packed_caps_far_above_the_scores(env, cap):
    """A cap's rounding goes by the score, not by the cap: the tolerance is that of calls without one."""
    lib, torch, _ = env
    torch.manual_seed(11)
    H, HKV, D, lens = 4, 2, 64, [300, 65]
    N = sum(lens)
    q, k, v = (torch.randn((N, h * D), device="cuda").half() for h in (H, HKV, HKV))
    cu = dev(torch, np.concatenate([[0], np.cumsum(lens)]).astype(np.int32))
    scale = 1.0 / np.sqrt(D)
    out = packed(env, "f16", q, k, v, cu, H, HKV, D, scale, cap)
    ref = packed64(torch, q, k, v, lens, H, HKV, D, scale, cap, 0)
    check_packed(host(out), *ref, H, D, "f16", 0.0, N)


def test_calls_side_by_side(env):
    """Calls of all three operators on two streams at once, each with a workspace and outputs of its own, leave what they
    leave alone."""
    lib, torch, _ = env
    H, HKV, D, n = 8, 2, 128, 4000
    c, *_ = filled(env, [n, n], HKV, D, seed=21)
    torch.manual_seed(21)
    lens = [700, 33, 0, 1200]
    N = sum(lens)
    cu = dev(torch, np.concatenate([[0], np.cumsum(lens)]).astype(np.int32))
    qp, kp, vp = (torch.randn((N, h * D), device="cuda").half() for h in (H, HKV, HKV))
    qt = [torch.randn((1, H * D), device="cuda").half() for _ in range(2)]
    seq, pos = [dev(torch, np.array([s], np.int32)) for s in range(2)], dev(torch, np.array([n - 1], np.int32))
    size = lib.fbx_kv4_attention_workspace(1, H, HKV, D, n)
    assert size > 0
    ws = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]

    def go(i, st, op, tok):
        assert lib.fbx_attention_packed(1, qp.data_ptr(), H * D, kp.data_ptr(), vp.data_ptr(), HKV * D, N, cu.data_ptr(), 4, H,
                                        HKV, D, 0.1, 0.0, 0, op.data_ptr(), H * D, st) == 0
        for _ in range(3):
            assert lib.fbx_kv4_attention(c.handle, 1, qt[i].data_ptr(), H * D, 1, H, seq[i].data_ptr(), pos.data_ptr(), n, 0.1,
                                         0.0, 0, tok.data_ptr(), H * D, ws[i].data_ptr(), size, st) == 0

    want = [(torch.zeros_like(qp), torch.zeros_like(qt[0])) for _ in range(2)]
    for i in range(2):
        go(i, None, *want[i])
    torch.cuda.synchronize()
    for _ in range(5):
        got = [(torch.zeros_like(qp), torch.zeros_like(qt[0])) for _ in range(2)]
        torch.cuda.synchronize()
        for i in range(2):
            go(i, streams[i].cuda_stream, *got[i])
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(got[i][0], want[i][0]) and torch.equal(got[i][1], want[i][1])
    assert int(c.err) == 0


def test_sequences_share_pages(env):
    """Two sequences whose tables name the same pages for a common prefix see the same keys there."""
    lib, torch, _ = env
    H, HKV, D = 4, 2, 96
    c, k, v, d, at = filled(env, [160, 160], HKV, D, seed=31)
    c.dtable[1, :8] = c.dtable[0, :8]
    q = torch.randn((1, H * D), device="cuda").expand(2, -1).contiguous()
    out = attention(env, c, "f32", q, H, [0, 1], [127, 127], 160, 0.1)
    assert torch.equal(out[0], out[1])
    out = attention(env, c, "f32", q, H, [0, 1], [159, 159], 160, 0.1)
    for s in range(2):
        rows = torch.cat([torch.arange(128), torch.arange(128, 160) + int(at[s])]).cuda()
        x, kk, vv, dd = q[s].view(HKV, 2, D).double(), *(y[rows].transpose(0, 1) for y in (k, v, d))
        w = torch.softmax(x @ kk.transpose(1, 2) * 0.1, -1)
        want, mean, coarse = (z.reshape(H, D).cpu().numpy() for z in (w @ vv, w @ vv.abs(), w @ dd))
        ext = (x.abs() @ kk.abs().transpose(1, 2)).amax(-1).reshape(H).cpu().numpy() * 0.1
        near(host(out[s]).reshape(H, D), want, (mean, ext, coarse), "f32")


@pytest.mark.parametrize("t,H,HKV,D,softcap,window", [("f16", 4, 4, 64, 0.0, 100), ("bf16", 4, 2, 96, 6.0, 0), ("f16", 8, 2, 128, 20.0, 65),
                                                      ("bf16", 12, 4, 128, 0.0, 64), ("f16", 10, 5, 96, 0.0, 1)])
def test_packed_many_short_prompts(env, t, H, HKV, D, softcap, window):
    """Batches of many short prompts, which take smaller key tiles: windows, caps, and values that are not finite."""
    lib, torch, _ = env
    torch.manual_seed(D + H)
    lens = many(6, 90, 0, 330) + [64, 65, 128, 1]
    N = sum(lens)
    q, k, v = (torch.randn((N, h * D), device="cuda").to(dtype(torch, t)) for h in (H, HKV, HKV))
    cu = dev(torch, np.concatenate([[0], np.cumsum(lens)]).astype(np.int32))
    scale = 1.3 / np.sqrt(D)
    clean = packed(env, t, q, k, v, cu, H, HKV, D, scale, softcap, window)
    check_packed(host(clean), *packed64(torch, q, k, v, lens, H, HKV, D, scale, softcap, window), H, D, t, softcap, N)
    ends = np.cumsum(lens)
    vv = v.clone()
    hit = torch.zeros_like(clean, dtype=torch.bool)
    for i, what in ((3, np.inf), (17, np.nan), (40, -np.inf), (91, np.inf)):
        n = lens[i]
        row = int(ends[i]) - n + n // 2
        vv[row, D - 1] = what          # kv head 0, its last dimension
        last = min(int(ends[i]), row + window) if window else int(ends[i])
        for h in range(H // HKV):
            hit[row:last, h * D + D - 1] = True
    out = packed(env, t, q, k, vv, cu, H, HKV, D, scale, softcap, window)
    assert torch.equal(out[~hit], clean[~hit]) and not bool(torch.isfinite(out[hit]).any())


# ------------------------------------------------------------------ values and scores at the edges


def appended(env, k, v):
    """One sequence's rows k, v [n][HKV][D] f32 appended without rotation: the cache, and what it holds, K, V and V's step (0
    where the stored d is not positive, whose codes are 0) in 64 bits."""
    lib, torch, _ = env
    n, HKV, D = k.shape
    c = Cache(env, [n], HKV, D, seed=n)
    x = dev(torch, np.concatenate([k.reshape(n, -1), v.reshape(n, -1)], 1).astype(np.float32))
    cos, sin = (dev(torch, a) for a in tables(n, 2))
    where = [dev(torch, a.astype(np.int32)) for a in (np.zeros(n), np.arange(n))]
    assert lib.fbx_kv4_append(c.handle, 0, None, x.data_ptr(), x.data_ptr() + 4 * HKV * D, 0, 2 * HKV * D, n, 0,
                              where[0].data_ptr(), where[1].data_ptr(), 0, 0, cos.data_ptr(), sin.data_ptr(), n, 0, None, 0, None,
                              None, 0, None) == 0
    torch.cuda.synchronize()
    held = [plain.values(*plain.quantise(y)).astype(np.float64) for y in (k, v)]
    step = np.maximum(plain.quantise(v)[1].astype(np.float64), 0.0).repeat(32, -1)
    return c, *held, step


def expect(q, k, v, step, H, scale, softcap=0.0):
    """plain.attend of one token's heads q [H][D] over all keys [n][HKV][D]: the result, mean, ext and coarse, heads first."""
    G = H // k.shape[1]
    parts = [plain.attend(q[h:h + 1], k[:, h // G], v[:, h // G], [len(k) - 1], scale, softcap, 0, step[:, h // G]) for h in range(H)]
    return [np.concatenate(x) for x in zip(*parts)]


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("value", [300.13, 1000.3, -300.07, 40.03, 65000.1, 1e-3, -2.0 ** -20 * 1.3])
def test_attention_over_groups_of_one_value(env, t, value):
    """A group of equal values that f16 does not hold: where f16 rounds the minimum up, the stored d is negative, all codes
    are 0, and the group stands for its lo. In every group, and beside groups of other sizes."""
    lib, torch, _ = env
    rng = np.random.default_rng(17)
    H, HKV, D, n = 8, 2, 128, 300
    k, v = (rng.standard_normal((n, HKV, D)).astype(np.float32) for _ in range(2))
    v[:, 0] = value
    v[:, 1, 32:64] = value
    v[n // 2:, 1, 96:] = value
    v[:, 1, 64:96] *= 1e-3
    c, kk, vv, step = appended(env, k, v)
    q = dev(torch, rng.standard_normal((1, H * D)).astype(np.float32), t)
    out = host(attention(env, c, t, q, H, [0], [n - 1], n, 0.1)).reshape(H, D)
    want, *size = expect(host(q).reshape(H, D).astype(np.float64), kk, vv, step, H, 0.1)
    near(out, want, size, t)


def outlier_slack(t, n, step):
    """What rounding to f16 may add for 16-bit types where the steps of a group lie far apart: a weight times its step is held to
    2^-25 of 2^(E - 7), 2^E the largest step's power of two, and meets codes of up to 15, against a sum of weights of 2 or
    more; n keys."""
    if t == "f32":
        return 0.0
    return n * 15 * 2.0 ** -26 * 2.0 ** (np.floor(np.log2(step.max(0))) - 7)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D", [64, 96, 128])
def test_attention_over_groups_far_apart(env, t, D):
    """V's groups of one head 2^12 to 2^22 apart: each keeps the precision that it has alone."""
    lib, torch, _ = env
    rng = np.random.default_rng(D)
    H, HKV, n = 4, 2, 200
    G, scale = H // HKV, 1.0 / np.sqrt(D)
    k, v = (rng.standard_normal((n, HKV, D)).astype(np.float32) for _ in range(2))
    sizes = np.array([2.0 ** 10, 2.0 ** -2, 2.0 ** -12, 2.0 ** -8])[:D // 32].repeat(32)
    c, kk, vv, step = appended(env, k, (v * sizes).astype(np.float32))
    q = dev(torch, rng.standard_normal((1, H * D)).astype(np.float32), t)
    out = host(attention(env, c, t, q, H, [0], [n - 1], n, scale)).reshape(H, D)
    want, *size = expect(host(q).reshape(H, D).astype(np.float64), kk, vv, step, H, scale)
    near(out, want, size, t)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("at", [0, 37, 59])
def test_attention_beside_a_key_of_huge_values(env, t, at):
    """One key whose V is 2^20 times the others' and whose weight is e^-64: it takes no bits from them."""
    lib, torch, _ = env
    rng = np.random.default_rng(at)
    H, D, n = 4, 128, 60
    k = np.zeros((n, 1, D), np.float32)
    v = np.tile(rng.standard_normal((1, 1, D)), (n, 1, 1)).astype(np.float32) * 2.0 ** -7
    k[at, 0, 0] = -64
    v[at] *= 2.0 ** 20
    c, kk, vv, step = appended(env, k, v)
    q = torch.zeros((1, H * D), device="cuda").to(dtype(torch, t))
    q.view(H, D)[:, 0] = 1.0
    out = host(attention(env, c, t, q, H, [0], [n - 1], n, 1.0)).reshape(H, D)
    want, mean, ext, coarse = expect(host(q).reshape(H, D).astype(np.float64), kk, vv, step, H, 1.0)
    # the outlier's own score is exact enough: its weight does not matter; the others' scores are 0
    tol = plain.allowed(want, mean, ext * 0, t, 2.0 ** -22 if t == "f32" else 2.0 ** -11, 0.0, coarse) + outlier_slack(t, n, step[:, 0])
    off = np.abs(out - want)
    assert (off <= tol).all(), (off / tol).max()


@pytest.mark.parametrize("t,size,scale,cap,n,H", [
    ("f32", 1e32, 0.1, 0.0, 1, 4), ("f32", 1e34, 0.1, 0.0, 600, 8), ("f32", 1e36, 0.5, 0.0, 3000, 1), ("f16", 1.0, 1e30, 0.0, 90, 8),
    ("bf16", 2.0 ** 110, 0.1, 0.0, 400, 8), ("bf16", 1e35, 0.5, 1e30, 600, 8), ("f16", 100.0, 1e29, 1e30, 33, 4),
])
def test_attention_of_scores_far_below_zero(env, t, size, scale, cap, n, H):
    """Scores that are finite, equal, and lower than -1e30: the weights are equal. One split, clusters, a second launch."""
    lib, torch, _ = env
    rng = np.random.default_rng(n)
    D = 128
    k = np.ones((n, 1, D), np.float32)
    v = rng.standard_normal((n, 1, D)).astype(np.float32)
    c, kk, vv, step = appended(env, k, v)
    q = torch.full((1, H * D), -size, device="cuda").to(dtype(torch, t))
    out = host(attention(env, c, t, q, H, [0], [n - 1], n, scale, cap)).reshape(H, D)
    want, mean, ext, coarse = expect(np.zeros((H, D)), kk, vv, step, H, 1.0)
    near(out, want, (mean, ext, coarse), t)


def test_host_arrays_are_refused_wherever_they_stand(env):
    """A host array in any place that is looked at: -1, and nothing is launched. Each place in turn, all others good; of the
    pairs the one that is looked at, and the other where it stands alone."""
    lib, torch, native = env
    H, HKV, D, n = 8, 2, 128, 64
    c = Cache(env, [n], HKV, D)
    keep = np.zeros(1 << 16, np.uint8)
    addr = (keep.ctypes.data + 15) // 16 * 16
    x = torch.randn((1, (H + 2 * HKV) * D), device="cuda")
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    cos, sin = (dev(torch, a) for a in tables(n, D))
    out = torch.full((3, H * D), 7.0, device="cuda")
    ws = torch.zeros(lib.fbx_kv4_attention_workspace(1, H, HKV, D, 1 << 17), dtype=torch.uint8, device="cuda")
    pool = c.pool.clone()

    def handle(**k):
        h = {f: getattr(c.handle, f) for f, _ in native.Kv4Cache._fields_}
        return native.Kv4Cache(**{**h, **k})

    def append(h=None, **k):
        p, ld = x.data_ptr(), x.shape[1]
        a = dict(type=0, q=p, k=p + 4 * H * D, v=p + 4 * (H + HKV) * D, ldq=ld, ldkv=ld, T=1, H=H, seq=zero.data_ptr(),
                 pos=zero.data_ptr(), rot=D, neox=0, cos=cos.data_ptr(), sin=sin.data_ptr(), n_rope=n, out=0, q_out=out.data_ptr(),
                 ldqo=H * D, k_out=out[1].data_ptr(), v_out=out[2].data_ptr(), ldkvo=HKV * D)
        a.update(k)
        return lib.fbx_kv4_append(h or c.handle, *a.values(), None)

    def attend(h=None, **k):
        a = dict(type=0, q=x.data_ptr(), ldq=H * D, T=1, H=H, seq=zero.data_ptr(), pos=zero.data_ptr(), keys=1 << 17, scale=0.1,
                 cap=0.0, window=0, out=out.data_ptr(), ldo=H * D, ws=ws.data_ptr(), size=ws.numel())
        a.update(k)
        return lib.fbx_kv4_attention(h or c.handle, *a.values(), None)

    assert ws.numel() > 0   # a second launch joins the splits
    for bad in ({"pool": addr}, {"page_table": addr}, {"err": addr}):
        assert append(handle(**bad)) == -1 and attend(handle(**bad)) == -1
    for bad in ({"q": addr}, {"k": addr}, {"pos": addr}, {"cos": addr}, {"q_out": addr}, {"k_out": addr},
                {"k_out": None, "v_out": addr}, {"k_out": addr, "v_out": None}):
        assert append(**bad) == -1
    for bad in ({"q": addr}, {"pos": addr}, {"out": addr}, {"ws": addr}):
        assert attend(**bad) == -1
    torch.cuda.synchronize()
    assert bool((out == 7).all()) and torch.equal(c.pool, pool)
    # each output of k and v alone
    assert append(k_out=None) == 0 and append(v_out=None) == 0
    assert append(handle(err=None), k_out=None, v_out=None) == 0 and attend(handle(err=None)) == 0
    torch.cuda.synchronize()


def rows64(torch, rows, q, k, v, H, HKV, D, scale, start=0):
    """packed64 of some rows (counted from their sequence's first row `start`)."""
    G = H // HKV
    want, mean, ext = [], [], []
    for r in rows:
        x = q[start + r].view(HKV, G, D).double()
        kk, vv = (y[start:start + r + 1].view(r + 1, HKV, D).transpose(0, 1).double() for y in (k, v))
        s = x @ kk.transpose(1, 2) * scale
        w = torch.softmax(s, -1)
        want.append((w @ vv).reshape(-1))
        mean.append((w @ vv.abs()).reshape(-1))
        ext.append((x.abs() @ kk.abs().transpose(1, 2)).amax(-1).reshape(-1) * scale)
    return [torch.stack(y).cpu().numpy() for y in (want, mean, ext)]


def test_packed_prompt_of_a_million_rows(env):
    """A job of 8192 key tiles, some 10 ms: the warps that wait for its end wait as long as it goes on."""
    lib, torch, _ = env
    n, D = (1 << 20) + 77, 64
    gen = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn((n, D), device="cuda", generator=gen).bfloat16() for _ in range(3))
    cu = dev(torch, np.array([0, n], np.int32))
    out = packed(env, "bf16", q, k, v, cu, 1, 1, D, 0.125)
    rows = [0, 1, 127, 128, 5000, n // 3, n // 2, n - 400, n - 130, n - 77, n - 2, n - 1]
    check_packed(host(out[rows]), *rows64(torch, rows, q, k, v, 1, 1, D, 0.125), 1, D, "bf16", 0.0, len(rows))
    assert bool(torch.isfinite(out).all())


@pytest.mark.parametrize("t,D,lens,window", [("bf16", 128, [40000, 700], 0), ("f16", 64, [33000, 100, 50], 0), ("f16", 128, [300, 36000, 9], 20000),
                                            ("bf16", 96, [3000] * 20, 1500)])
def test_packed_infinities_in_long_prompts(env, t, D, lens, window):
    """An infinity or NaN near the end of a long prompt, and a sequence of NaN behind it: rows that do not see them keep every
    bit, rows that do are not finite in that dimension alone."""
    lib, torch, _ = env
    H, HKV = 4, 2
    N, ends = sum(lens), np.cumsum(lens)
    s = int(np.argmax(lens))
    a, z = int(ends[s]) - lens[s], int(ends[s])
    gen = torch.Generator(device="cuda").manual_seed(D)
    q, k, v = (torch.randn((N, w * D), device="cuda", generator=gen).to(dtype(torch, t)) for w in (H, HKV, HKV))
    cu = dev(torch, np.concatenate([[0], ends]).astype(np.int32))
    clean = packed(env, t, q, k, v, cu, H, HKV, D, 0.1, 0.0, window)
    assert bool(torch.isfinite(clean).all())
    for row, what in ((z - 1, np.inf), (z - 200, -np.inf), (z - 333, np.nan), (a + 5, np.inf)):
        vv = v.clone()
        vv[row, D + 7] = what          # kv head 1, dimension 7
        vv[z:] = np.nan                # every later sequence
        out = packed(env, t, q, k, vv, cu, H, HKV, D, 0.1, 0.0, window)
        hit = torch.zeros_like(out, dtype=torch.bool)
        for h in (2, 3):
            hit[row:min(z, row + window) if window else z, h * D + 7] = True
        hit[z:] = True
        assert torch.equal(out[~hit], clean[~hit]) and not bool(torch.isfinite(out[hit]).any())


def test_packed_prompt_of_nan_values(env):
    """Every value of one kv head NaN: its heads give NaN, the others what they give without."""
    lib, torch, _ = env
    n, H, HKV, D = 9000, 4, 2, 128
    q, k, v = (torch.randn((n, w * D), device="cuda").half() for w in (H, HKV, HKV))
    cu = dev(torch, np.array([0, 4000, n], np.int32))
    clean = packed(env, "f16", q, k, v, cu, H, HKV, D, 0.1)
    v[:, :D] = np.nan
    out = packed(env, "f16", q, k, v, cu, H, HKV, D, 0.1)
    assert bool(torch.isnan(out[:, :2 * D]).all()) and torch.equal(out[:, 2 * D:], clean[:, 2 * D:])


def test_packed_one_key_above_thousands(env):
    """One key 17.5 nats above all others, with a V of 0: what the row gives is the others', whose weights are 2^-25 each."""
    lib, torch, _ = env
    n, H, D = 8192, 2, 64
    for t in ("f16", "bf16"):
        q, k = (torch.zeros((n, w * D), device="cuda").to(dtype(torch, t)) for w in (H, 1))
        v = torch.rand((n, D), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).to(dtype(torch, t)) + 0.5
        q[:, ::D] = 1.0
        k[0, 0] = 17.5
        v[0] = 0
        cu = dev(torch, np.array([0, n], np.int32))
        out = packed(env, t, q, k, v, cu, H, 1, D, 1.0)
        want, mean, ext = packed64(torch, q, k, v, [n], H, 1, D, 1.0, 0.0, 0)
        # products of 17.5 and 1 and sums with zeros are exact; the weight, once rounded, carries the exponential's error alone
        check_packed(host(out), want, mean, ext * 0, H, D, t, 0.0, n)


@pytest.mark.parametrize("t,H,HKV", [("f16", 14, 2), ("bf16", 6, 2), ("f16", 50, 1)])
def test_packed_groups_that_leave_rows_over(env, t, H, HKV):
    """Groups that do not divide a tile's 128 rows leave some that are nobody's, and hold what an earlier call left there: NaN
    does not reach the others."""
    lib, torch, _ = env
    D, n = 128, 900
    gen = torch.Generator(device="cuda").manual_seed(H)
    q, k, v = (torch.randn((n, w * D), device="cuda", generator=gen).to(dtype(torch, t)) for w in (H, HKV, HKV))
    cu = dev(torch, np.array([0, 333, n], np.int32))
    clean = packed(env, t, q, k, v, cu, H, HKV, D, 0.1)
    check_packed(host(clean), *packed64(torch, q, k, v, [333, n - 333], H, HKV, D, 0.1, 0.0, 0), H, D, t, 0.0, n)
    nan = torch.full((20000, 4 * D), float("nan"), device="cuda", dtype=q.dtype)
    bad = packed(env, t, nan, nan[:, :D].contiguous(), nan[:, :D].contiguous(), dev(torch, np.array([0, 20000], np.int32)), 4, 1, D, 0.1)
    assert bool(torch.isnan(bad).all())
    assert torch.equal(packed(env, t, q, k, v, cu, H, HKV, D, 0.1), clean)


def test_append_without_rotation_needs_no_tables(env):
    """rot 0: no table, no bound on positions from one, the same cache and outputs as with tables."""
    lib, torch, _ = env
    H, HKV, D, T = 4, 2, 128, 70
    qkv = torch.randn((T, (H + 2 * HKV) * D), device="cuda")
    cos, sin = (dev(torch, x) for x in tables(T, 2))
    a, b = (Cache(env, [T], HKV, D, seed=1) for _ in range(2))
    rc, q_out, k_out, v_out = call_append(env, a, "f32", qkv, H, [0] * T, list(range(T)), 0, False, cos, sin, "f32")
    assert rc == 0
    got = [torch.zeros_like(x) for x in (q_out, k_out, v_out)]
    where = [dev(torch, x.astype(np.int32)) for x in (np.zeros(T), np.arange(T))]
    x, ld = qkv.data_ptr(), qkv.shape[1]
    for n_rope in (1, 0):
        assert lib.fbx_kv4_append(b.handle, 0, x, x + 4 * H * D, x + 4 * (H + HKV) * D, ld, ld, T, H, where[0].data_ptr(),
                                  where[1].data_ptr(), 0, 1, None, None, n_rope, 0, got[0].data_ptr(), H * D, got[1].data_ptr(),
                                  got[2].data_ptr(), HKV * D, None) == 0
        torch.cuda.synchronize()
        assert int(b.err) == 0 and torch.equal(a.pool, b.pool)
        assert all(torch.equal(x, y) for x, y in zip(got, (q_out, k_out, v_out)))


# more heads than the warps of a CTA have in one turn: type, out, T, lens, H, HKV, D, rot, neox, layers, layer
APPENDS_OF_SEVERAL_TURNS = [
    ("f16", "f16", 150, [150], 28, 4, 128, 128, True, 1, 0),
    ("bf16", "bf16", 149, [149], 64, 8, 128, 128, False, 1, 0),
    ("f16", "f32", 148, [148], 90, 3, 128, 128, False, 1, 0),     # more than five turns of 16 heads: fetched again
    ("f32", "f32", 148, [148], 40, 4, 128, 128, False, 1, 0),     # more than two
    ("f32", "bf16", 148, [148], 40, 4, 128, 20, True, 1, 0),
    ("bf16", "f16", 148, [148], 33, 4, 96, 96, True, 1, 0),       # a ragged last turn, 8 lanes of a warp idle
    ("bf16", "f16", 148, [148], 85, 2, 96, 32, False, 1, 0),
    ("f16", "bf16", 148, [148], 37, 3, 64, 22, True, 1, 0),
    ("bf16", "bf16", 148, [148], 160, 4, 64, 64, True, 1, 0),
]


@pytest.mark.parametrize("case", APPENDS_OF_SEVERAL_TURNS, ids=lambda c: "-".join(map(str, c[:9])))
def test_append_of_many_heads_matches_the_format(env, case):
    test_append_matches_the_format_bit_for_bit(env, *case)


@pytest.mark.parametrize("t,H,HKV,D,rot,neox", [("bf16", 64, 8, 128, 128, True), ("f16", 90, 3, 128, 64, False), ("f32", 40, 4, 96, 20, True),
                                               ("f16", 28, 4, 128, 128, True), ("f32", 40, 4, 128, 128, False)])
def test_append_of_many_heads_in_place(env, t, H, HKV, D, rot, neox):
    lib, torch, _ = env
    T = 160
    cos, sin = (dev(torch, x) for x in tables(T, rot))
    seq, pos = dev(torch, np.zeros(T, np.int32)), dev(torch, np.arange(T, dtype=np.int32))
    qkv = torch.randn((T, (H + 2 * HKV) * D), device="cuda").to(dtype(torch, t))
    a, b = (Cache(env, [T], HKV, D, seed=1) for _ in range(2))
    rc, *want = call_append(env, a, t, qkv, H, [0] * T, list(range(T)), rot, neox, cos, sin, t)
    assert rc == 0
    x, ld, es = qkv.clone(), qkv.shape[1], qkv.element_size()
    p = [x.data_ptr() + es * D * o for o in (0, H, H + HKV)]
    assert lib.fbx_kv4_append(b.handle, plain.TYPE[t], *p, ld, ld, T, H, seq.data_ptr(), pos.data_ptr(), rot, int(neox), cos.data_ptr(),
                              sin.data_ptr(), T, plain.TYPE[t], p[0], ld, p[1], p[2], ld, None) == 0
    torch.cuda.synchronize()
    assert torch.equal(x, torch.cat(want, 1)) and torch.equal(a.pool, b.pool)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_attention_of_a_token_alone_and_among_others(env, t):
    """How a context is split goes by the whole call, and a row's last bits with it: alone it is as near to 64 bits as among
    others, and the same call gives the same bits."""
    lib, torch, _ = env
    H, HKV, D, lens = 8, 2, 128, [2000, 333, 40, 1] * 12
    c, k, v, d, at = filled(env, lens, HKV, D, seed=41)
    T = len(lens)
    q = torch.randn((T, H * D), device="cuda", generator=torch.Generator(device="cuda").manual_seed(41)).to(dtype(torch, t))
    together = attention(env, c, t, q, H, list(range(T)), [n - 1 for n in lens], max(lens), 0.1)
    assert torch.equal(together, attention(env, c, t, q, H, list(range(T)), [n - 1 for n in lens], max(lens), 0.1))
    for s in (0, 1, 2, 3, T - 4):
        alone = attention(env, c, t, q[s:s + 1], H, [s], [lens[s] - 1], lens[s], 0.1)[0]
        rows = slice(int(at[s]), int(at[s]) + lens[s])
        x = q[s].view(HKV, H // HKV, D).double()
        kk, vv, dd = (y[rows].transpose(0, 1) for y in (k, v, d))
        w = torch.softmax(x @ kk.transpose(1, 2) * 0.1, -1)
        want, mean, coarse = (z.reshape(H, D).cpu().numpy() for z in (w @ vv, w @ vv.abs(), w @ dd))
        ext = (x.abs() @ kk.abs().transpose(1, 2)).amax(-1).reshape(H).cpu().numpy() * 0.1
        for got in (alone, together[s]):
            near(host(got).reshape(H, D), want, (mean, ext, coarse), t)
    assert int(c.err) == 0


@pytest.mark.parametrize("count", [200, 1 << 20])
def test_packed_lengths_that_go_back_and_forth(env, count):
    """Lengths that name the same rows again and again (which the caller must not give): as much work as proper ones can be,
    inside the buffers; a proper call after it is right."""
    lib, torch, _ = env
    H, HKV, D, N = 2, 1, 64, 20000
    gen = torch.Generator(device="cuda").manual_seed(8)
    q, k, v = (torch.randn((N, w * D), device="cuda", generator=gen).half() for w in (H, HKV, HKV))
    cu = torch.zeros(count + 1, dtype=torch.int32, device="cuda")
    cu[1::2] = N
    guard = torch.full((N + 256, H * D), 7.0, device="cuda", dtype=torch.float16)
    t = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
    t[0].record()
    packed(env, "f16", q, k, v, cu, H, HKV, D, 0.1, out=guard[128:128 + N])
    t[1].record()
    torch.cuda.synchronize()
    # at most N / 128 + min(count, N) jobs, each of at most N / 64 key tiles of some 2 us on one of 148 SMs: 0.1 s; times 20
    assert t[0].elapsed_time(t[1]) < 2000
    assert bool((guard[:128] == 7).all()) and bool((guard[128 + N:] == 7).all()) and bool(torch.isfinite(guard).all())
    cu = dev(torch, np.array([0, 300, 800], np.int32))
    out = packed(env, "f16", q[:800], k[:800], v[:800], cu, H, HKV, D, 0.1)
    check_packed(host(out), *packed64(torch, q[:800], k[:800], v[:800], [300, 500], H, HKV, D, 0.1, 0.0, 0), H, D, "f16", 0.0, 800)


@pytest.mark.parametrize("D", [64, 128])
def test_packed_between_matrix_products(env, D):
    """Packed attention in a row with matrix products, which use tensor memory too, eager and captured: each gets what it needs,
    whichever begins early."""
    lib, torch, _ = env
    H, HKV, lens = 16, 4, [500, 3, 700]
    N = sum(lens)
    gen = torch.Generator(device="cuda").manual_seed(D)
    q, k, v = (torch.randn((N, w * D), device="cuda", generator=gen).bfloat16() for w in (H, HKV, HKV))
    w = (torch.randn((H * D, H * D), device="cuda", generator=gen) * (H * D) ** -0.5).bfloat16()
    cu = dev(torch, np.concatenate([[0], np.cumsum(lens)]).astype(np.int32))
    outs = [torch.zeros((N, H * D), device="cuda", dtype=q.dtype) for _ in range(4)]

    def chain(st):
        x = q
        for out in outs:
            assert lib.fbx_attention_packed(30, x.data_ptr(), H * D, k.data_ptr(), v.data_ptr(), HKV * D, N, cu.data_ptr(), 3, H, HKV,
                                            D, 0.1, 0.0, 0, out.data_ptr(), H * D, st) == 0
            x = torch.matmul(out, w)
        return x

    want = chain(None).clone()
    kept = [o.clone() for o in outs]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain(torch.cuda.current_stream().cuda_stream)
    for _ in range(10):
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(outs, kept))
    check_packed(host(outs[0]), *packed64(torch, q, k, v, lens, H, HKV, D, 0.1, 0.0, 0), H, D, "bf16", 0.0, N)


@pytest.mark.parametrize("t,apart", [("f32", 12), ("f16", 20), ("bf16", 20)])
def test_attention_of_queries_far_apart(env, t, apart):
    """Queries of one group 2^apart below another's, and keys as much above: both have the same part in the scores."""
    lib, torch, _ = env
    rng = np.random.default_rng(apart)
    H, HKV, D, n = 4, 2, 128, 200
    k, v = (rng.standard_normal((n, HKV, D)).astype(np.float32) for _ in range(2))
    size = np.array([0, apart, apart // 2, apart], np.float64).repeat(32)   # binary orders
    k = (k * 2.0 ** (size - apart // 2)).astype(np.float32)
    c, kk, vv, step = appended(env, k, v)
    q = dev(torch, (rng.standard_normal((1, H * D)) * np.tile(2.0 ** (apart // 2 - size), H)).astype(np.float32), t)
    out = host(attention(env, c, t, q, H, [0], [n - 1], n, 0.1)).reshape(H, D)
    want, *bound = expect(host(q).reshape(H, D).astype(np.float64), kk, vv, step, H, 0.1)
    near(out, want, bound, t)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_attention_of_many_tokens_over_one_long_context(env, t):
    """131000 keys that no call splits, as there are tokens enough: 16000 a warp, V's values all of one sign."""
    lib, torch, _ = env
    n, T, H, D = 131000, 300, 8, 64
    c = Cache(env, [n], 1, D, seed=1)
    gen = torch.Generator(device="cuda").manual_seed(n)
    x = torch.cat([torch.randn((n, D), device="cuda", generator=gen),
                   torch.empty((n, D), device="cuda").exponential_(generator=gen)], 1).contiguous()
    held = [torch.empty((n, D), device="cuda") for _ in range(2)]
    where = [torch.zeros(n, dtype=torch.int32, device="cuda"), torch.arange(n, dtype=torch.int32, device="cuda")]
    assert lib.fbx_kv4_append(c.handle, 0, None, x.data_ptr(), x.data_ptr() + 4 * D, 0, 2 * D, n, 0, where[0].data_ptr(),
                              where[1].data_ptr(), 0, 0, None, None, 0, 0, None, 0, held[0].data_ptr(), held[1].data_ptr(), D,
                              None) == 0
    q = torch.randn((T, H * D), device="cuda", generator=gen).to(dtype(torch, t))
    out = attention(env, c, t, q, H, [0] * T, [n - 1] * T, n, 0.1)
    k, v = (y.double() for y in held)
    y = x[:, D:].view(n, D // 32, 32)
    d = ((y.amax(-1) - y.amin(-1)) / 15 * 1.001).double().repeat_interleave(32, -1)   # no less than the d that is stored
    for r in (0, 150, T - 1):
        a = q[r].view(H, D).double()
        w = torch.softmax(a @ k.T * 0.1, -1)
        want, mean, coarse = ((w @ z).cpu().numpy() for z in (v, v, d))
        ext = (a.abs() @ k.abs().T).amax(-1).cpu().numpy() * 0.1
        near(host(out[r]).reshape(H, D), want, (mean, ext, coarse), t)


@pytest.mark.parametrize("t,D,n", [("f16", 64, 131072), ("f16", 96, 100000), ("f16", 128, 131072), ("bf16", 128, 131072), ("f16", 64, 1 << 20)])
def test_packed_long_prompts_of_one_sign(env, t, D, n):
    """Values around 1, so that every key adds to the accumulator: it loses nothing on the way that the sum of the weights keeps."""
    lib, torch, _ = env
    gen = torch.Generator(device="cuda").manual_seed(n + D)
    q, k, v = (torch.randn((n, D), device="cuda", generator=gen) for _ in range(3))
    q, k, v = (x.to(dtype(torch, t)) for x in (q, k, 1 + 0.1 * v))
    cu = dev(torch, np.array([0, n], np.int32))
    out = packed(env, t, q, k, v, cu, 1, 1, D, D ** -0.5)
    rows = [0, 777, 16384, n // 3, n // 2, n - 100, n - 2, n - 1]
    check_packed(host(out[rows]), *rows64(torch, rows, q, k, v, 1, 1, D, D ** -0.5), 1, D, t, 0.0, len(rows))


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 96, 128])
def test_attention_rounds_a_weight_once(env, t, D):
    """Contexts of a few keys and many heads, whose outputs are often much smaller than the values: what is left there is the
    rounding of a weight times its step, once."""
    lib, torch, _ = env
    H, HKV, lens = 160, 8, [2, 3, 2, 5, 1, 13, 2, 388] * 12
    for seed in range(4):
        c, k, v, d, at = filled(env, lens, HKV, D, seed=100 + seed, spread=20.0 + seed)
        T = len(lens)
        q = (torch.randn((T, H * D), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)) / 20).to(dtype(torch, t))
        out = host(attention(env, c, t, q, H, list(range(T)), [n - 1 for n in lens], max(lens), D ** -0.5))
        for s in range(T):
            rows = slice(int(at[s]), int(at[s]) + lens[s])
            x = q[s].view(HKV, H // HKV, D).double()
            kk, vv, dd = (y[rows].transpose(0, 1) for y in (k, v, d))
            w = torch.softmax(x @ kk.transpose(1, 2) * D ** -0.5, -1)
            want, mean, coarse = (z.reshape(H, D).cpu().numpy() for z in (w @ vv, w @ vv.abs(), w @ dd))
            ext = (x.abs() @ kk.abs().transpose(1, 2)).amax(-1).reshape(H).cpu().numpy() * D ** -0.5
            near(out[s].reshape(H, D), want, (mean, ext, coarse), t)
