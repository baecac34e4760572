"""Refusals of the device-buffer entry points (no device needed: the arguments
are looked at first), and the plain forms that the GPU tests compare with."""
from __future__ import annotations

import numpy as np
import pytest

import kv4_plain as plain


@pytest.fixture(scope="module")
def lib():
    from imurun_b200 import native
    return native.load_library()


def cache(**k):
    from imurun_b200 import native
    a = dict(pool=4096, page_table=4096, err=None, page_stride=5120, layer_offset=0, n_pages=4, table_stride=4, n_seqs=2,
             n_head_kv=2, head_dim=128)
    return native.Kv4Cache(**{**a, **k})


def append(lib, c=None, **k):
    a = dict(type=0, q=4096, k=4096 * 2, v=4096 * 3, ldq=512, ldkv=256, T=1, H=4, seq=4096, pos=4096, rot=128, neox=0,
             cos=4096, sin=4096, n_rope=10, out_type=1, q_out=4096 * 4, ldqo=512, k_out=None, v_out=None, ldkvo=0)
    a.update(k)
    return lib.fbx_kv4_append(c or cache(), *a.values(), None)


def attend(lib, c=None, **k):
    a = dict(type=0, q=4096, ldq=512, T=1, H=4, seq=4096, pos=4096, max_keys=10, scale=0.1, softcap=0.0, window=0, out=8192,
             ldo=512, ws=4096, ws_bytes=1 << 30)
    a.update(k)
    return lib.fbx_kv4_attention(c or cache(), *a.values(), None)


def packed(lib, **k):
    a = dict(type=1, q=4096, ldq=512, k=8192, v=8192, ldkv=256, rows=10, cu=4096, B=2, H=4, HKV=2, D=128, scale=0.1,
             softcap=0.0, window=0, out=4096, ldo=512)
    a.update(k)
    return lib.fbx_attention_packed(*a.values(), None)


BAD_CACHES = [dict(pool=None), dict(page_table=None), dict(pool=4100), dict(head_dim=80), dict(n_head_kv=0), dict(n_pages=0),
              dict(table_stride=0), dict(n_seqs=0), dict(page_stride=5104), dict(page_stride=5128), dict(layer_offset=16),
              dict(layer_offset=-16), dict(layer_offset=8, page_stride=1 << 20), dict(page_stride=-5120)]


def test_good_arguments_pass_the_checks(lib):
    """With no device they get as far as asking for one; fake addresses are no device memory where there is one."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("addresses that are no memory")
    assert append(lib) > 0 and attend(lib) > 0 and packed(lib) > 0
    assert append(lib, q=None, q_out=None, ldq=0, ldqo=0) > 0
    assert append(lib, rot=0, cos=None, sin=None) > 0
    assert append(lib, T=0) == 0 and attend(lib, T=0) == 0 and packed(lib, rows=0) == 0


@pytest.mark.parametrize("bad", BAD_CACHES)
def test_caches_that_cannot_be_are_refused(lib, bad):
    assert append(lib, cache(**bad)) == -1 and attend(lib, cache(**bad)) == -1


def test_no_cache_is_refused(lib):
    assert lib.fbx_kv4_append(None, *([0] * 2), None, None, *([0] * 4), *([None] * 2), 0, 0, None, None, 0, 0, None, 0, None,
                              None, 0, None) == -1


@pytest.mark.parametrize("bad", [dict(type=8), dict(type=2), dict(out_type=12), dict(T=-1), dict(k=None), dict(v=None),
                                 dict(seq=None), dict(pos=None), dict(q=None), dict(q_out=None), dict(rot=130), dict(rot=3),
                                 dict(rot=-2), dict(n_rope=0), dict(cos=None), dict(sin=None), dict(H=0), dict(ldq=508),
                                 dict(ldq=513), dict(ldkv=252), dict(ldqo=500), dict(ldqo=516), dict(q=4100), dict(k=4104),
                                 dict(v=4097), dict(q_out=4098), dict(k_out=8, ldkvo=256), dict(k_out=4096, ldkvo=0),
                                 dict(v_out=4096, ldkvo=255), dict(q_out=4096), dict(k_out=8192, ldkvo=256),
                                 dict(type=0, out_type=0, q_out=4096, ldqo=1024), dict(H=70000)])
def test_append_refuses(lib, bad):
    assert append(lib, **bad) == -1


@pytest.mark.parametrize("bad", [dict(type=12), dict(T=-1), dict(T=70000), dict(q=None), dict(out=None), dict(seq=None),
                                 dict(pos=None), dict(max_keys=0), dict(H=0), dict(H=5), dict(ldq=511), dict(ldq=514),
                                 dict(ldo=100), dict(softcap=-1.0), dict(softcap=float("nan")), dict(scale=float("nan")), dict(scale=-1.0),
                                 dict(window=-1), dict(q=4100), dict(out=4100), dict(ws=4100)])
def test_attention_refuses(lib, bad):
    assert attend(lib, **bad) == -1


def test_attention_refuses_a_small_workspace(lib):
    for T, keys in ((1, 577), (1, 131071), (64, 2180), (3, 1)):
        need = lib.fbx_kv4_attention_workspace(T, 4, 2, 128, keys)
        if need:
            assert attend(lib, T=T, max_keys=keys, ws_bytes=need - 1) == -1 and attend(lib, T=T, max_keys=keys, ws=None) == -1
    assert lib.fbx_kv4_attention_workspace(0, 4, 2, 128, 10) == 0 and lib.fbx_kv4_attention_workspace(1, 5, 2, 128, 10) == 0


@pytest.mark.parametrize("bad", [dict(type=0), dict(type=8), dict(q=None), dict(k=None), dict(v=None), dict(out=None),
                                 dict(cu=None), dict(rows=-1), dict(B=0), dict(B=-2), dict(H=0), dict(HKV=0), dict(H=5),
                                 dict(D=80), dict(D=256), dict(ldq=504), dict(ldq=516), dict(ldkv=248), dict(ldkv=260),
                                 dict(ldo=511), dict(softcap=-0.5), dict(scale=float("nan")), dict(scale=0.0), dict(scale=float("inf")), dict(H=258, ldq=33024, ldo=33024), dict(window=-3), dict(q=4100),
                                 dict(k=4104), dict(v=8), dict(out=4097)])
def test_packed_refuses(lib, bad):
    assert packed(lib, **bad) == -1


def test_layer_bytes(lib):
    for D in (64, 96, 128):
        assert lib.fbx_kv4_layer_bytes(3, D) == 3 * plain.record_bytes(D)
    assert lib.fbx_kv4_layer_bytes(0, 128) == 0 and lib.fbx_kv4_layer_bytes(1, 256) == 0


@pytest.mark.parametrize("D", [64, 96, 128])
def test_format_holds_every_value_once(D):
    """Every (row, dimension) has a nibble of its own, and what is stored comes back."""
    for row in range(16):
        for where in (lambda d: plain.k_byte(D, d), lambda d: plain.v_byte(D, d, row)):
            assert len({(where(d), d & 1) for d in range(D)}) == D and max(where(d) for d in range(D)) == D // 2 - 1
    rng = np.random.default_rng(D)
    pool = np.full(3 * plain.record_bytes(D), 0xEE, np.uint8)
    x = rng.standard_normal((16, 2, D)).astype(np.float32)
    for row in range(16):
        for is_v in (0, 1):
            plain.store(pool, plain.record_bytes(D), row, is_v, D, *plain.quantise(x[row, is_v][None]))
    assert (pool[:plain.record_bytes(D)] == 0xEE).all() and (pool[2 * plain.record_bytes(D):] == 0xEE).all()
    k, v = plain.fetch(pool, plain.record_bytes(D), D)
    for got, want in ((k, x[:, 0]), (v, x[:, 1])):
        codes, d, lo = plain.quantise(want)
        assert np.array_equal(got.astype(np.float32), plain.values(codes, d, lo))
        # half a code of the group's range, and the rounding of lo and d to f16
        assert (np.abs(got - want).reshape(16, -1, 32) <= 0.5 * d[..., None].astype(np.float64) + 2e-2).all()


def test_empty_calls_need_no_buffers(lib):
    assert append(lib, T=0, k=None, v=None, q=None, q_out=None, seq=None, pos=None) == 0
    assert attend(lib, T=0, q=None, out=None, seq=None, pos=None) == 0
    assert packed(lib, rows=0, q=None, k=None, v=None, out=None) == 0


@pytest.mark.parametrize("bad", [dict(softcap=1e-31), dict(scale=1e20, softcap=1e-15), dict(scale=2e30), dict(softcap=2e30)])
def test_scales_that_could_overflow_are_refused(lib, bad):
    assert attend(lib, **bad) == -1 and packed(lib, **bad) == -1


@pytest.mark.parametrize("off", [1, 2, 3])
def test_arrays_of_32_bit_values_off_their_boundary_are_refused(lib, off):
    """Sequences, positions, tables, the page table, the error word and the lengths: an unaligned load would fault."""
    at = 4096 + off
    for bad in (dict(seq=at), dict(pos=at), dict(cos=at), dict(sin=at)):
        assert append(lib, **bad) == -1
    for bad in (dict(seq=at), dict(pos=at)):
        assert attend(lib, **bad) == -1
    for bad in (dict(page_table=at), dict(err=at)):
        assert append(lib, cache(**bad)) == -1 and attend(lib, cache(**bad)) == -1
    assert packed(lib, cu=at) == -1


def test_append_without_rotation_asks_for_no_tables(lib):
    import torch
    if torch.cuda.is_available():
        pytest.skip("addresses that are no memory")
    assert append(lib, rot=0, n_rope=0) > 0 and append(lib, rot=0, n_rope=-1, cos=None, sin=3) > 0
    assert append(lib, rot=2, n_rope=0) == -1 and append(lib, rot=2, n_rope=-1) == -1
