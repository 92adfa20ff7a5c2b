"""Refusals and argument plumbing of the 8-bit cache's calls, on the CPU: the public
functions with the device predicate patched and nothing launched, and the C entry
points' own checks, which come before any launch."""
from __future__ import annotations

import ctypes
import os

import pytest
import torch

import mtlflashattn_amd as mfa
from mtlflashattn_amd import _build, _hip, _kernel

F8 = torch.float8_e4m3fn


def t(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


def i32(*x):
    return torch.tensor(x, dtype=torch.int32)


def caches(P=2, page=64, H=2, D=64):
    return (mfa.kv8_cache(P, page, H, D, device="cpu") for _ in range(2))


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_build.LIB_PATH):
        _build.build()
    return _hip.load()


@pytest.fixture
def launches(monkeypatch):
    """(name, parameters) of every launch; CPU tensors count as ROCm tensors."""
    calls = []
    monkeypatch.setattr(_kernel, "_is_rocm_tensor", lambda x: True)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 0, raising=False)
    for name in ("kv8_append", "kv8_fwd", "kv8_weights", "kv8_evict"):
        monkeypatch.setattr(_hip, name, lambda *a, name=name: calls.append((name, a[0])))
    for name in ("kv8_fwd_workspace_bytes", "kv8_evict_workspace_bytes"):
        monkeypatch.setattr(_hip, name, lambda p: 0)
    return calls


def test_cache_shapes():
    codes, scales = mfa.kv8_cache(3, 128, 2, 96, device="cpu")
    assert codes.shape == (3, 128, 2, 96) and codes.dtype == F8 and scales.shape == (3, 2, 2) and scales.dtype == torch.uint8
    assert codes.stride() == (2 * 128 * 96, 96, 128 * 96, 1) and scales.stride() == (4, 1, 2)
    assert not codes.float().any() and not scales.any()
    for page, D, exc in ((32, 64, ValueError), (0, 64, ValueError), (64, 80, NotImplementedError), (64, 160, NotImplementedError)):
        with pytest.raises(exc):
            mfa.kv8_cache(2, page, 2, D, device="cpu")


def test_cpu_tensors_raise():
    kc, vc = caches()
    table, w = i32(1)[None], torch.zeros(2, 64, 2)
    for call in (lambda: mfa.kv8_append(t(1, 2, 64), t(1, 2, 64), kc, vc, i32(0, 1), i32(0), table),
                 lambda: mfa.flash_attn_kv8_func(t(1, 1, 2, 64), kc, vc, i32(3), table),
                 lambda: mfa.kv8_key_weights(t(1, 1, 2, 64), kc, torch.zeros(1, 2, 1), w, i32(3), table),
                 lambda: mfa.kv8_evict(kc, vc, w, i32(3), table, 2, 1)):
        with pytest.raises(NotImplementedError, match="ROCm GPU only"):
            call()


def bad_caches():
    kc, _ = caches()
    return [dict(cache=None), dict(cache=kc[0]), dict(cache=(kc[0],)), dict(cache=(kc[0], None)), dict(cache=(kc[0].view(torch.uint8), kc[1])),
            dict(cache=(kc[0], kc[1].float())), dict(cache=(kc[0], kc[1][:, :, :1])), dict(cache=(kc[0], kc[1][..., None])),
            dict(cache=(kc[0][:, :32], kc[1])), dict(cache=(kc[0][0], kc[1])), dict(cache=tuple(caches(page=128))[0]),
            dict(cache=tuple(caches(H=4))[0]), dict(cache=(t(2, 64, 2, 128, dtype=torch.uint8).view(F8)[..., ::2], kc[1])),
            dict(cache=(t(2, 64, 2, 72, dtype=torch.uint8).view(F8)[..., :64], kc[1])), dict(cache=mfa.kv4_cache(2, 64, 2, 64, device="cpu"))]


@pytest.mark.parametrize("i", range(15))
@pytest.mark.parametrize("which", ["k_cache", "v_cache"])
def test_bad_caches(launches, i, which):
    cache = bad_caches()[i]["cache"]
    kc, vc = caches()
    table, w = i32(1)[None], torch.zeros(2, 64, 2)
    both = dict(k_cache=kc, v_cache=vc)
    both[which] = cache
    refused = (ValueError, NotImplementedError)
    with pytest.raises(refused):
        mfa.kv8_append(t(1, 2, 64), t(1, 2, 64), both["k_cache"], both["v_cache"], i32(0, 1), i32(0), table)
    with pytest.raises(refused):
        mfa.flash_attn_kv8_func(t(1, 1, 4, 64), both["k_cache"], both["v_cache"], i32(3), table)
    with pytest.raises(refused):
        mfa.kv8_evict(both["k_cache"], both["v_cache"], w, i32(3), table, 2, 1)
    if which == "k_cache":
        with pytest.raises(refused):
            mfa.kv8_key_weights(t(1, 1, 4, 64), cache, torch.zeros(1, 4, 1), w, i32(3), table)
    assert not launches


@pytest.mark.parametrize("change,exc", [
    (dict(k=t(2, 64)), ValueError), (dict(v=t(3, 2, 64)), ValueError), (dict(v=t(2, 2, 64, dtype=torch.float16)), NotImplementedError),
    (dict(k=t(2, 2, 64, dtype=torch.int32), v=t(2, 2, 64, dtype=torch.int32)), NotImplementedError),
    (dict(k=t(2, 2, 80), v=t(2, 2, 80)), NotImplementedError), (dict(k=t(2, 4, 64), v=t(2, 4, 64)), ValueError),
    (dict(cu_seqlens=i32(0, 1)), ValueError), (dict(cache_seqlens=torch.zeros(2)), ValueError),
    (dict(cache_seqlens=i32(0)), ValueError), (dict(block_table=i32(1)[None]), ValueError),
    (dict(block_table=i32(1, 2)), ValueError), (dict(block_table=torch.zeros(2, 1, dtype=torch.int64)), ValueError),
    (dict(block_table=torch.zeros(2, 4, dtype=torch.int32)[:, ::2]), ValueError), (dict(cu_seqlens=None), ValueError),
    (dict(k=t(2, 2, 64).requires_grad_()), NotImplementedError),
])
def test_append(launches, change, exc):
    kc, vc = caches()
    good = dict(k=t(2, 2, 64), v=t(2, 2, 64), k_cache=kc, v_cache=vc, cu_seqlens=i32(0, 1, 2), cache_seqlens=i32(0, 3),
                block_table=torch.zeros(2, 1, dtype=torch.int32))
    with pytest.raises(exc):
        mfa.kv8_append(**{**good, **change})
    assert not launches
    versions = [x._version for c in (kc, vc) for x in c]
    mfa.kv8_append(**good)
    assert len(launches) == 1 and all(x._version > v for x, v in zip((*kc, *vc), versions))


@pytest.mark.parametrize("change,exc", [
    (dict(q=t(2, 4, 64)), ValueError), (dict(q=t(2, 1, 3, 64)), ValueError),
    (dict(q=t(2, 1, 4, 64, dtype=torch.float32)), NotImplementedError), (dict(q=t(2, 1, 4, 80)), NotImplementedError),
    (dict(q=t(2, 1, 4, 128)), ValueError), (dict(cache_seqlens=i32(1)), ValueError),
    (dict(block_table=i32(1)[None]), ValueError), (dict(window_size=(-2, 0)), ValueError), (dict(window_size=3), ValueError),
    (dict(softcap=-1.0), ValueError), (dict(alibi_slopes=[0.5]), TypeError), (dict(alibi_slopes=torch.zeros(3)), ValueError),
    (dict(max_seqlen_k=-1), ValueError), (dict(q=t(2, 1, 4, 64).requires_grad_()), NotImplementedError),
    (dict(cache_seqlens=[1, 2]), ValueError), (dict(block_table=None), ValueError),
])
def test_attend_and_weights(launches, change, exc):
    kc, vc = caches()
    good = dict(q=t(2, 1, 4, 64), k_cache=kc, cache_seqlens=i32(0, 3), block_table=torch.zeros(2, 1, dtype=torch.int32))
    more = dict(softmax_lse=torch.zeros(2, 4, 1), weights=torch.zeros(2, 64, 2))
    with pytest.raises(exc):
        mfa.flash_attn_kv8_func(**{**good, **change}, v_cache=vc)
    with pytest.raises(exc):
        mfa.kv8_key_weights(**{**good, **change}, **more)
    assert not launches
    mfa.flash_attn_kv8_func(**good, v_cache=vc)
    version = more["weights"]._version
    mfa.kv8_key_weights(**good, **more)
    assert [n for n, _ in launches] == ["kv8_fwd", "kv8_weights"] and more["weights"]._version > version


@pytest.mark.parametrize("change,exc", [
    (dict(softmax_lse=torch.zeros(2, 1, 4)), ValueError), (dict(softmax_lse=t(2, 4, 1)), ValueError), (dict(softmax_lse=None), ValueError),
    (dict(weights=t(2, 64, 2)), ValueError), (dict(weights=torch.zeros(2, 64, 4)), ValueError), (dict(weights=torch.zeros(3, 64, 2)), ValueError),
    (dict(weights=torch.zeros(1, 64, 2).expand(2, 64, 2)), ValueError), (dict(weights=None), ValueError),
    (dict(weights=torch.zeros(2, 64, 2).requires_grad_()), NotImplementedError),
    (dict(softmax_lse=torch.zeros(2, 4, 1).requires_grad_()), NotImplementedError),
    (dict(cu_seqlens_q=i32(0, 1, 2)), ValueError), (dict(q=t(2, 4, 64), cu_seqlens_q=i32(0, 2), softmax_lse=torch.zeros(4, 2)), ValueError),
])
def test_weights(launches, change, exc):
    kc, _ = caches()
    good = dict(q=t(2, 1, 4, 64), k_cache=kc, cache_seqlens=i32(0, 3), block_table=torch.zeros(2, 1, dtype=torch.int32),
                softmax_lse=torch.zeros(2, 4, 1), weights=torch.zeros(2, 64, 2))
    with pytest.raises(exc):
        mfa.kv8_key_weights(**{**good, **change})
    assert not launches
    mfa.kv8_key_weights(**{**good, "q": t(2, 4, 64), "cu_seqlens_q": i32(0, 1, 2), "softmax_lse": torch.zeros(4, 2)})
    assert len(launches) == 1


@pytest.mark.parametrize("change,exc", [
    (dict(weights=t(2, 64, 2)), ValueError), (dict(weights=torch.zeros(2, 64, 4)), ValueError), (dict(weights=None), ValueError),
    (dict(weights=torch.zeros(2, 64, 1).expand(2, 64, 2)), ValueError), (dict(weights=torch.zeros(2, 64, 2).requires_grad_()), NotImplementedError),
    (dict(cache_seqlens=i32(1)), ValueError), (dict(cache_seqlens=torch.zeros(2)), ValueError), (dict(cache_seqlens=[1, 2]), ValueError),
    (dict(block_table=i32(1)[None]), ValueError), (dict(budget=-1), ValueError), (dict(recent=-1), ValueError),
    (dict(max_seqlen_k=-1), ValueError),
])
def test_evict(launches, change, exc):
    kc, vc = caches()
    good = dict(k_cache=kc, v_cache=vc, weights=torch.zeros(2, 64, 2), cache_seqlens=i32(0, 3),
                block_table=torch.zeros(2, 1, dtype=torch.int32), budget=2, recent=1)
    with pytest.raises(exc):
        mfa.kv8_evict(**{**good, **change})
    assert not launches
    versions = [x._version for x in (*kc, *vc, good["weights"])]
    out = mfa.kv8_evict(**good)
    assert out.shape == (2,) and out.dtype == torch.int32 and len(launches) == 1
    assert all(x._version > v for x, v in zip((*kc, *vc, good["weights"]), versions))
    for which in (0, 1):
        e = tuple(x[:1].expand(2, *x.shape[1:]) if i == which else x for i, x in enumerate(kc))
        for a, b in ((e, vc), (vc, e)):
            with pytest.raises(ValueError, match="expanded"):
                mfa.kv8_evict(**{**good, "k_cache": a, "v_cache": b})
            with pytest.raises(ValueError, match="expanded"):
                mfa.kv8_append(t(3, 2, 64), t(3, 2, 64), a, b, i32(0, 3), i32(0), i32(0, 1)[None])


def test_strides_reach_the_library(launches):
    kc, vc = caches(P=4, page=128, H=2, D=64)
    table = torch.zeros(2, 5, dtype=torch.int32)[:, :3]
    w = torch.zeros(4, 2, 128).transpose(1, 2)
    q = t(2, 3, 8, 64)[:, :, 2:6]
    mfa.flash_attn_kv8_func(q, kc, vc, i32(0, 3), table, window_size=[7, -1], causal=True, softcap=2.0)
    mfa.kv8_key_weights(q, kc, torch.zeros(2, 4, 3), w, i32(0, 3), table, window_size=[7, -1], causal=True, softcap=2.0)
    mfa.kv8_evict(kc, vc, w, i32(0, 3), table, 1 << 40, 5, max_seqlen_k=1 << 50)
    (_, p), (_, kw), (_, ev) = launches
    for c in (p.cache, ev.cache):
        assert (c.k.code_page_stride, c.k.code_row_stride, c.k.code_head_stride) == (2 * 128 * 64, 64, 128 * 64)
        assert (c.v.scale_page_stride, c.v.scale_row_stride, c.v.scale_head_stride) == (2 * 2, 1, 2)
        assert (c.max_pages, c.page_block_size, c.num_pages, c.block_table_batch_stride) == (3, 128, 4, 5)
    for f in (p, kw.fwd):
        assert (f.q_batch_stride, f.q_seq_stride, f.q_head_stride) == (3 * 8 * 64, 8 * 64, 64)
        assert (f.window_left, f.window_right, f.causal, f.max_seqlen_k, f.softcap) == (7, -1, 1, 384, 2.0)
        assert abs(f.scale - 0.125) < 1e-7
    assert (kw.fwd.lse_batch_stride, kw.fwd.lse_head_stride) == (12, 3)
    for x in (kw, ev):
        assert (x.weight_page_stride, x.weight_row_stride, x.weight_head_stride) == (256, 1, 128)
    assert (ev.budget, ev.recent, ev.max_seqlen_k) == (2 ** 31 - 1, 5, 384)


def test_numbers_given_as_tensors_are_read_at_every_call(launches):
    kc, vc = caches()
    scale, budget = torch.tensor(0.5), torch.tensor(1)
    q, table, w = t(1, 1, 2, 64), i32(0, 1)[None], torch.zeros(2, 64, 2)
    for s, n in ((0.5, 1), (0.25, 7)):
        scale.fill_(s)
        budget.fill_(n)
        mfa.flash_attn_kv8_func(q, kc, vc, i32(5), table, softmax_scale=scale)
        mfa.kv8_key_weights(q, kc, torch.zeros(1, 2, 1), w, i32(5), table, softmax_scale=scale)
        mfa.kv8_evict(kc, vc, w, i32(5), table, budget, budget)
        assert launches[-3][1].scale == s and launches[-2][1].fwd.scale == s and launches[-1][1].budget == n


def test_forward_mode_derivatives_are_refused(launches):
    import torch.autograd.forward_ad as fw

    kc, vc = caches()
    q, table, w, lse = t(1, 3, 2, 64), i32(0, 1)[None], torch.zeros(2, 64, 2), torch.zeros(1, 2, 3)
    with fw.dual_level():
        dual = lambda x: fw.make_dual(x, torch.ones_like(x))  # noqa: E731
        for call in (lambda: mfa.flash_attn_kv8_func(dual(q), kc, vc, i32(5), table),
                     lambda: mfa.kv8_append(dual(q)[0], q[0], kc, vc, i32(0, 3), i32(0), table),
                     lambda: mfa.kv8_key_weights(dual(q), kc, lse, w, i32(5), table),
                     lambda: mfa.kv8_key_weights(q, kc, dual(lse), w, i32(5), table),
                     lambda: mfa.kv8_evict(kc, vc, dual(w), i32(5), table, 2, 1)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
    assert not launches


@pytest.mark.parametrize("rows", [1 << 31, 1 << 40])
def test_sizes_beyond_32_bits(launches, rows):
    kc, vc = caches()
    table = i32(0)[None].expand(1, rows // 64)
    w = torch.zeros(2, 64, 2)
    for call in (lambda: mfa.flash_attn_kv8_func(t(1, 1, 2, 64), kc, vc, i32(3), table),
                 lambda: mfa.kv8_append(t(3, 2, 64), t(3, 2, 64), kc, vc, i32(0, 3), i32(0), table),
                 lambda: mfa.kv8_evict(kc, vc, w, i32(3), table, 2, 1)):
        with pytest.raises(ValueError):
            call()
    assert not launches


# --------------------------------------------------------------------------
# the C entry points


def refused(lib, rc, code, text):
    assert rc == code and text in lib.mfa_last_error().decode()


def cache_params(cache, D=64, Hkv=2):
    for pool in (cache.k, cache.v):
        pool.codes = pool.scales = 4096
        pool.code_page_stride, pool.code_row_stride, pool.code_head_stride = Hkv * 64 * D, D, 64 * D
        pool.scale_page_stride, pool.scale_row_stride, pool.scale_head_stride = Hkv, 1, 1
    cache.block_table = 4096
    cache.max_pages, cache.page_block_size, cache.num_pages = 4, 64, 8


def fwd_params(D=64, H=4, Hkv=2, p=None):
    p = _hip.MfaKv4FwdParams() if p is None else p
    cache_params(p.cache, D, Hkv)
    p.q = p.o = p.cache_seqlens = 4096
    p.q_batch_stride = p.o_batch_stride = p.q_seq_stride = p.o_seq_stride = H * D
    p.q_head_stride = p.o_head_stride = D
    p.batch, p.seqlen_q, p.heads_q, p.heads_kv, p.head_dim = 2, 1, H, Hkv, D
    p.scale = 0.125
    p.window_left = p.window_right = -1
    p.dtype = _hip.MFA_DTYPE_BF16
    return p


FWD = [
    (lambda p: setattr(p, "dtype", 2), -2, "dtype"), (lambda p: setattr(p, "head_dim", 80), -2, "head_dim"),
    (lambda p: setattr(p, "batch", -1), -1, "negative"), (lambda p: setattr(p, "heads_kv", 3), -1, "divide"),
    (lambda p: setattr(p, "softcap", float("nan")), -1, "softcap"), (lambda p: setattr(p, "window_left", -2), -1, "window"),
    (lambda p: setattr(p, "q", 4098), -1, "aligned"), (lambda p: setattr(p, "cache_seqlens", None), -1, "cache_seqlens"),
    (lambda p: setattr(p, "q_head_stride", 4), -1, "strides"), (lambda p: setattr(p, "seqlen_q", 1 << 30), -1, "too large"),
    (lambda p: setattr(p.cache, "page_block_size", 32), -1, "page_block_size"),
    (lambda p: setattr(p.cache, "block_table", None), -1, "block_table"), (lambda p: setattr(p.cache, "max_pages", 1 << 30), -1, "2^31"),
    (lambda p: setattr(p.cache.k, "codes", 4100), -1, "codes"), (lambda p: setattr(p.cache.k, "code_row_stride", 8), -1, "16 bytes"),
    (lambda p: setattr(p.cache.k, "scale_row_stride", -1), -1, ">= 0"), (lambda p: setattr(p.cache.k, "code_row_stride", 1 << 30), -1, "2 GiB"),
]


@pytest.mark.parametrize("change,code,text", FWD)
def test_c_attend_and_weights(lib, change, code, text):
    p = fwd_params()
    assert lib.mfa_kv8_fwd_workspace_bytes(ctypes.byref(p)) > 0
    change(p)
    refused(lib, lib.mfa_kv8_fwd(ctypes.byref(p), None, 0, None), code, text)
    assert "mfa_kv8_fwd" in lib.mfa_last_error().decode()
    refused(lib, lib.mfa_kv8_fwd_workspace_bytes(ctypes.byref(p)), code, text)
    w = weights_params()
    change(w.fwd)
    refused(lib, lib.mfa_kv8_weights(ctypes.byref(w), None), code, text)


def weights_params():
    w = _hip.MfaKv8WeightsParams()
    fwd_params(p=w.fwd)
    w.fwd.softmax_lse = w.weights = 4096
    w.weight_page_stride, w.weight_row_stride, w.weight_head_stride = 128, 1, 64
    return w


def test_c_weights(lib):
    for change, text in ((lambda w: setattr(w.fwd, "softmax_lse", None), "softmax_lse"), (lambda w: setattr(w, "weights", 4098), "weights"),
                         (lambda w: setattr(w, "weights", None), "weights"), (lambda w: setattr(w, "weight_row_stride", -1), ">= 0"),
                         (lambda w: setattr(w, "weight_row_stride", 1 << 28), "2 GiB")):
        w = weights_params()
        change(w)
        refused(lib, lib.mfa_kv8_weights(ctypes.byref(w), None), -1, text)
    refused(lib, lib.mfa_kv8_weights(None, None), -1, "NULL")
    for field in ("batch", "seqlen_q"):
        w = weights_params()
        setattr(w.fwd, field, 0)
        assert lib.mfa_kv8_weights(ctypes.byref(w), None) == 0


def test_c_attend_workspace(lib):
    p = fwd_params()
    need = lib.mfa_kv8_fwd_workspace_bytes(ctypes.byref(p))
    refused(lib, lib.mfa_kv8_fwd(ctypes.byref(p), None, need, None), -1, "workspace")
    refused(lib, lib.mfa_kv8_fwd(ctypes.byref(p), 4096 + 16, need, None), -1, "aligned")
    refused(lib, lib.mfa_kv8_fwd(ctypes.byref(p), 4096, need - 1, None), -1, "needed")
    refused(lib, lib.mfa_kv8_fwd(None, None, 0, None), -1, "NULL")
    p.batch = 0
    assert lib.mfa_kv8_fwd(ctypes.byref(p), None, 0, None) == 0


def test_c_append(lib):
    def params():
        p = _hip.MfaKv4AppendParams()
        cache_params(p.cache)
        p.k = p.v = p.cu_seqlens = p.cache_seqlens = 4096
        p.k_token_stride = p.v_token_stride = 128
        p.k_head_stride = p.v_head_stride = 64
        p.batch, p.total, p.heads_kv, p.head_dim, p.dtype = 2, 5, 2, 64, 1
        return p
    for change, code, text in (
            (dict(dtype=3), -1, "dtype"), (dict(total=-1), -1, "negative"), (dict(head_dim=72), -2, "head_dim"),
            (dict(k=4098), -1, "aligned"), (dict(v_token_stride=4), -1, "strides"), (dict(k_values=4096), -1, "values"),
            (dict(cu_seqlens=None), -1, "cu_seqlens"), (dict(total=1 << 30), -1, "too large")):
        p = params()
        for k, v in change.items():
            setattr(p, k, v)
        refused(lib, lib.mfa_kv8_append(ctypes.byref(p), None), code, text)
    p = params()
    p.total = 0
    assert lib.mfa_kv8_append(ctypes.byref(p), None) == 0
    refused(lib, lib.mfa_kv8_append(None, None), -1, "NULL")


def test_c_evict(lib):
    def params():
        p = _hip.MfaKv8EvictParams()
        cache_params(p.cache)
        p.weights = p.cache_seqlens = p.new_seqlens = 4096
        p.weight_page_stride, p.weight_row_stride, p.weight_head_stride = 128, 1, 64
        p.batch, p.heads_kv, p.head_dim, p.budget, p.recent = 2, 2, 64, 100, 10
        return p
    need = lib.mfa_kv8_evict_workspace_bytes(ctypes.byref(params()))
    assert need >= 2 * 2 * 100 * (2 * 64 + 10)
    for change, code, text in (
            (dict(head_dim=72), -2, "head_dim"), (dict(batch=-1), -1, "negative"), (dict(budget=-1), -1, "negative"),
            (dict(recent=-1), -1, "negative"), (dict(heads_kv=0), -1, "heads"), (dict(cache_seqlens=None), -1, "cache_seqlens"),
            (dict(new_seqlens=4097), -1, "new_seqlens"), (dict(weights=None), -1, "weights"), (dict(weight_head_stride=-1), -1, ">= 0"),
            (dict(batch=1 << 30), -1, "too large")):
        p = params()
        for k, v in change.items():
            setattr(p, k, v)
        refused(lib, lib.mfa_kv8_evict(ctypes.byref(p), None, 0, None), code, text)
        refused(lib, lib.mfa_kv8_evict_workspace_bytes(ctypes.byref(p)), code, text)
    p = params()
    for change in (dict(budget=0), dict(budget=256), dict(max_seqlen_k=100), dict(max_seqlen_k=7)):  # (no row moves)
        p = params()
        for k, v in change.items():
            setattr(p, k, v)
        assert lib.mfa_kv8_evict_workspace_bytes(ctypes.byref(p)) == 0
    p = params()
    p.cache.num_pages = (1 << 31) // p.cache.page_block_size
    refused(lib, lib.mfa_kv8_evict_workspace_bytes(ctypes.byref(p)), -1, "2^31 - 1 rows")
    p = params()
    refused(lib, lib.mfa_kv8_evict(ctypes.byref(p), None, need, None), -1, "workspace")
    refused(lib, lib.mfa_kv8_evict(ctypes.byref(p), 4096 + 16, need, None), -1, "aligned")
    refused(lib, lib.mfa_kv8_evict(ctypes.byref(p), 4096, need - 1, None), -1, "needed")
    refused(lib, lib.mfa_kv8_evict(ctypes.byref(p), 4096, need, None), -1, "same memory")
    refused(lib, lib.mfa_kv8_evict(None, None, 0, None), -1, "NULL")
    p.batch = 0
    assert lib.mfa_kv8_evict(ctypes.byref(p), None, 0, None) == 0
