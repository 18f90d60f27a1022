"""CPU: what the C entry points of the transformer layers refuse, before anything is launched, and what is nothing to do."""
import ctypes as C

import pytest

from tensor_amd import capi

P = 4096  # an address that nothing reads


@pytest.fixture(scope="module")
def lib():
    L = capi.load_cdll()
    L.otter_hip_last_error.restype = C.c_char_p
    for f in ("otter_hip_kv_page_bytes", "otter_hip_kv_attend_workspace_bytes", "otter_hip_linear_workspace_bytes"):
        getattr(L, f).restype = C.c_size_t
    return L


def cache(**kw):
    return capi.KvCacheArgs(**dict(dict(heads=2, head_dim=64, n_pages=8, keys=P, values=P, key_scales=P, value_scales=P), **kw))


def batch(**kw):
    return capi.KvBatchArgs(**dict(dict(n_seqs=2, n_tokens=4, max_pages=3, starts=P, lengths=P, pages=P), **kw))


def desc(**kw):
    return capi.KvAttendDesc(**dict(dict(q_heads=4, scale=1.0, cap=0.0, causal=1, window=0, slopes=None), **kw))


def calls(L, c, b, d):
    at = lambda s: C.byref(s) if s is not None else None
    n, v = C.c_size_t(128), C.c_void_p(P)
    return [L.otter_hip_kv_append(at(c), at(b), v, n, v, n, None), L.otter_hip_kv_read(at(c), at(b), v, v, None),
            L.otter_hip_kv_attend(at(c), at(b), at(d), v, n, v, v, C.c_size_t(1 << 40), None)]


@pytest.mark.parametrize("kw", [dict(heads=0), dict(head_dim=0), dict(head_dim=257), dict(n_pages=0), dict(keys=None), dict(values=None),
                                dict(key_scales=None), dict(value_scales=None), dict(keys=P + 8), dict(values=P + 1), dict(heads=1 << 20)])
def test_caches(lib, kw):
    assert all(rc in (-1, -2) for rc in calls(lib, cache(**kw), batch(), desc()))
    assert lib.otter_hip_last_error()
    assert calls(lib, None, batch(), desc()) == [-2] * 3


@pytest.mark.parametrize("kw", [dict(n_seqs=-1), dict(n_tokens=-1), dict(max_pages=-1), dict(starts=None), dict(lengths=None), dict(pages=None),
                                dict(n_seqs=1 << 21), dict(max_pages=1 << 25), dict(n_seqs=1 << 20, heads=4096), dict(n_tokens=1 << 27, heads=4),
                                dict(n_tokens=2 ** 31 - 1, heads=256)])
def test_batches(lib, kw):
    c = cache(heads=kw.pop("heads", 2))
    assert all(rc in (-1, -2) for rc in calls(lib, c, batch(**kw), desc(q_heads=c.heads)))
    assert calls(lib, cache(), None, desc()) == [-2] * 3


@pytest.mark.parametrize("kw", [dict(q_heads=0), dict(q_heads=3), dict(scale=float("nan")), dict(scale=float("inf")), dict(cap=-1.0),
                                dict(cap=float("nan")), dict(cap=1e-39, scale=3e38), dict(cap=3e38), dict(scale=-3e38), dict(window=-1), dict(q_heads=1 << 30)])
def test_attention(lib, kw):
    assert calls(lib, cache(), batch(), desc(**kw))[2] in (-1, -2)
    assert lib.otter_hip_kv_attend_workspace_bytes(C.byref(cache()), C.byref(batch()), C.byref(desc(**kw))) == 0
    assert calls(lib, cache(), batch(), None)[2] == -2


def test_attention_needs_its_workspace(lib):
    c, b, d = cache(), batch(n_seqs=1, n_tokens=1, max_pages=1000), desc()
    need = lib.otter_hip_kv_attend_workspace_bytes(C.byref(c), C.byref(b), C.byref(d))
    assert need > 0
    v, n = C.c_void_p(P), C.c_size_t(256)
    for work, size in ((None, need), (P, need - 1), (P + 4, need)):
        assert lib.otter_hip_kv_attend(C.byref(c), C.byref(b), C.byref(d), v, n, v, C.c_void_p(work), C.c_size_t(size), None) == -2
    for q, out in ((None, v), (v, None)):
        assert lib.otter_hip_kv_attend(C.byref(c), C.byref(b), C.byref(d), q, n, out, v, C.c_size_t(need), None) == -2
    assert lib.otter_hip_kv_append(C.byref(c), C.byref(b), None, n, v, n, None) == -2


@pytest.mark.parametrize("kw", [dict(n_seqs=0), dict(n_tokens=0), dict(n_seqs=0, starts=None, lengths=None, pages=None)])
def test_nothing_to_do(lib, kw):
    assert calls(lib, cache(), batch(**kw), desc()) == [0, 0, 0]


@pytest.mark.parametrize("heads,dim,pages", [(1, 1, 4096), (1, 64, 4096), (2, 65, 16384), (8, 128, 65536), (1, 256, 16384), (0, 64, 0), (1, 257, 0),
                                             (1, 0, 0)])
def test_page_bytes(lib, heads, dim, pages):
    assert lib.otter_hip_kv_page_bytes(heads, dim) == pages


@pytest.mark.parametrize("kw", [dict(experts=0), dict(in_features=0), dict(out_features=0), dict(in_features=131073), dict(gated=2),
                                dict(activation_type=6), dict(activation_type=-1), dict(gated=1, activation_type=1), dict(experts=1 << 17),
                                dict(experts=1 << 16, out_features=1 << 24, in_features=64)])
def test_layers(lib, kw):
    d = capi.LinearDesc(**dict(dict(experts=1, in_features=64, out_features=16, gated=0, activation_type=0), **kw))
    h = C.c_void_p(1)
    assert lib.otter_hip_linear_create(C.byref(d), C.c_void_p(P), C.c_void_p(P), None, C.byref(h)) in (-1, -2)
    assert not h.value


def test_layers_without_a_part(lib):
    d, h, v = capi.LinearDesc(1, 64, 16, 0, 0, 0.0), C.c_void_p(), C.c_void_p(P)
    assert lib.otter_hip_linear_create(None, v, v, None, C.byref(h)) == -2
    assert lib.otter_hip_linear_create(C.byref(d), None, v, None, C.byref(h)) == -2
    assert lib.otter_hip_linear_create(C.byref(d), v, None, None, C.byref(h)) == -2
    assert lib.otter_hip_linear_create(C.byref(d), v, v, None, None) == -2
    assert lib.otter_hip_linear_forward(None, v, C.c_size_t(64), 1, None, None, 1, v, v, C.c_size_t(1 << 20), None) == -2
    assert lib.otter_hip_linear_workspace_bytes(None, 1, 1) == 0
    assert lib.otter_hip_linear_kernel_kind(None, 1) == -2 and lib.otter_hip_linear_set_kernel(None, 0) == -2
    assert lib.otter_hip_linear_destroy(None) == 0
