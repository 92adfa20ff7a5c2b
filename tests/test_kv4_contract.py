"""Refusals of the operators around the attention call, on the CPU: the public
functions' argument checks with the device predicate patched and nothing launched,
and the C entry points' own checks, which come before any launch."""
from __future__ import annotations

import ctypes
import os

import pytest
import torch

import mtlflashattn_amd as mfa
from mtlflashattn_amd import _build, _hip, _kernel


def t(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


def i32(*x):
    return torch.tensor(x, dtype=torch.int32)


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_build.LIB_PATH):
        _build.build()
    return _hip.load()


@pytest.fixture
def launches(monkeypatch):
    """Treat CPU tensors as ROCm tensors and count launches instead of making them."""
    calls = []
    monkeypatch.setattr(_kernel, "_is_rocm_tensor", lambda x: True)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 0, raising=False)
    for name in ("norm_rope", "kv4_append", "kv4_fwd", "copy_pages"):
        monkeypatch.setattr(_hip, name, lambda *a, name=name: calls.append((name, a)))
    monkeypatch.setattr(_hip, "kv4_fwd_workspace_bytes", lambda p: 0)
    return calls


def test_cpu_tensors_raise():
    c = mfa.kv4_cache(2, 64, 2, 64, device="cpu")
    with pytest.raises(NotImplementedError, match="ROCm GPU only"):
        mfa.qk_norm_rope(t(4, 2, 64), t(4, 2, 64), None, None, t(8, 32), t(8, 32))
    with pytest.raises(NotImplementedError, match="ROCm GPU only"):
        mfa.kv4_append(t(1, 2, 64), t(1, 2, 64), c, c, i32(0, 1), i32(0), i32(1)[None])
    with pytest.raises(NotImplementedError, match="ROCm GPU only"):
        mfa.flash_attn_kv4_func(t(1, 1, 2, 64), c, c, i32(3), i32(1)[None])
    with pytest.raises(NotImplementedError, match="ROCm GPU only"):
        mfa.copy_cache_pages([t(4, 8)], i32(0), i32(1))


class TestNormRope:
    good = dict(q=t(2, 5, 4, 64), k=t(2, 5, 2, 64), q_weight=t(64), k_weight=t(64), cos=t(9, 32, dtype=torch.float32),
                sin=t(9, 32, dtype=torch.float32), positions=torch.zeros(2, 5, dtype=torch.int32))

    @pytest.mark.parametrize("change,exc", [
        (dict(q=t(5, 4, 64)), ValueError), (dict(q=t(2, 4, 4, 64)), ValueError), (dict(k=t(2, 5, 2, 32)), ValueError),
        (dict(q=t(4, 64), k=t(2, 64)), ValueError), (dict(k=t(2, 5, 2, 64, dtype=torch.float16)), NotImplementedError),
        (dict(q=t(2, 5, 4, 64, dtype=torch.float64), k=t(2, 5, 2, 64, dtype=torch.float64)), NotImplementedError),
        (dict(q=t(2, 5, 4, 136), k=t(2, 5, 2, 136)), NotImplementedError),
        (dict(q_weight=t(32)), ValueError), (dict(k_weight=t(64, dtype=torch.float32)), ValueError),
        (dict(q_weight=t(64, dtype=torch.int32)), ValueError), (dict(cos=t(9, 16, dtype=torch.float32)), ValueError),
        (dict(cos=t(9, 32), sin=t(9, 32, dtype=torch.float32)), ValueError),
        (dict(cos=t(9, 33, dtype=torch.float32), sin=t(9, 33, dtype=torch.float32)), ValueError),
        (dict(cos=t(9, 32, dtype=torch.float16), sin=t(9, 32, dtype=torch.float16)), ValueError),
        (dict(positions=torch.zeros(2, 5)), ValueError), (dict(positions=torch.zeros(2, dtype=torch.int32)), ValueError),
        (dict(positions=[0, 1, 2, 3, 4]), ValueError), (dict(eps=-1.0), ValueError), (dict(eps=float("nan")), ValueError),
        (dict(cos=t(9, 32, dtype=torch.float32).requires_grad_()), NotImplementedError),
        (dict(q=[1.0]), ValueError),
    ])
    def test_refusals(self, launches, change, exc):
        with pytest.raises(exc):
            mfa.qk_norm_rope(**{**self.good, **change})
        assert not launches

    def test_strides_reach_the_library(self, launches):
        qkv = t(2, 5, 8, 64)
        mfa.qk_norm_rope(**{**self.good, "q": qkv[:, :, :4], "k": qkv[:, :, 4:6]}, interleaved=True, eps=1e-5)
        p = launches[-1][1][0]
        assert (p.q_batch_stride, p.q_seq_stride, p.q_head_stride) == (5 * 8 * 64, 8 * 64, 64)
        assert (p.batch, p.seqlen, p.heads_q, p.heads_kv, p.head_dim, p.rotary_dim, p.table_rows) == (2, 5, 4, 2, 64, 64, 9)
        assert p.interleaved == 1 and p.positions_batch_stride == 5 and p.positions_64 == 0
        assert p.dtype_weight == _hip.MFA_DTYPE_BF16 and p.dtype_table == _hip.MFA_DTYPE_F32


def caches(P=4, page=64, H=2, D=64):
    return mfa.kv4_cache(P, page, H, D, device="cpu"), mfa.kv4_cache(P, page, H, D, device="cpu")


@pytest.mark.parametrize("page,D,exc", [(0, 64, ValueError), (-64, 64, ValueError), (32, 64, ValueError),
                                        (100, 64, ValueError), (64, 80, NotImplementedError), (64, 0, NotImplementedError),
                                        (64, 160, NotImplementedError)])
def test_cache_sizes(page, D, exc):
    with pytest.raises(exc):
        mfa.kv4_cache(4, page, 2, D, device="cpu")


def bad_caches():
    (codes, scales), _ = caches()
    return [
        codes, (codes,), (codes, None), (codes.float(), scales), (codes, scales.float()), (codes[0], scales[0]),
        (codes[:, :32], scales[:, :32]), (codes[:3], scales), (codes[..., :16], scales), (codes, scales[..., :1]),
        (codes[:, :, :1], scales[:, :, :1]),
        (torch.zeros(4, 64, 2, 64, dtype=torch.uint8)[..., ::2], scales),
        (torch.zeros(4, 64, 2, 40, dtype=torch.uint8)[..., :32], scales),
    ]


class TestCacheArguments:
    @pytest.mark.parametrize("i", range(13))
    def test_bad_caches(self, launches, i):
        good, bad = caches()[0], bad_caches()[i]
        for kc, vc in ((good, bad), (bad, good)):
            with pytest.raises(ValueError):
                mfa.kv4_append(t(1, 2, 64), t(1, 2, 64), kc, vc, i32(0, 1), i32(0), i32(1)[None])
            with pytest.raises(ValueError):
                mfa.flash_attn_kv4_func(t(1, 1, 4, 64), kc, vc, i32(3), i32(1)[None])
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
    def test_append(self, launches, change, exc):
        kc, vc = caches()
        good = dict(k=t(2, 2, 64), v=t(2, 2, 64), k_cache=kc, v_cache=vc, cu_seqlens=i32(0, 1, 2), cache_seqlens=i32(0, 3),
                    block_table=torch.zeros(2, 1, dtype=torch.int32))
        with pytest.raises(exc):
            mfa.kv4_append(**{**good, **change})
        assert not launches
        mfa.kv4_append(**good)
        assert len(launches) == 1

    @pytest.mark.parametrize("change,exc", [
        (dict(q=t(2, 4, 64)), ValueError), (dict(q=t(2, 1, 3, 64)), ValueError),
        (dict(q=t(2, 1, 4, 64, dtype=torch.float32)), NotImplementedError), (dict(q=t(2, 1, 4, 80)), NotImplementedError),
        (dict(q=t(2, 1, 4, 128)), ValueError), (dict(cache_seqlens=i32(1)), ValueError),
        (dict(block_table=i32(1)[None]), ValueError), (dict(window_size=(-2, 0)), ValueError), (dict(window_size=3), ValueError),
        (dict(softcap=-1.0), ValueError), (dict(alibi_slopes=[0.5]), TypeError), (dict(alibi_slopes=torch.zeros(3)), ValueError),
        (dict(max_seqlen_k=-1), ValueError), (dict(q=t(2, 1, 4, 64).requires_grad_()), NotImplementedError),
        (dict(cache_seqlens=[1, 2]), ValueError), (dict(block_table=None), ValueError),
    ])
    def test_attend(self, launches, change, exc):
        kc, vc = caches()
        good = dict(q=t(2, 1, 4, 64), k_cache=kc, v_cache=vc, cache_seqlens=i32(0, 3),
                    block_table=torch.zeros(2, 1, dtype=torch.int32))
        with pytest.raises(exc):
            mfa.flash_attn_kv4_func(**{**good, **change})
        assert not launches
        mfa.flash_attn_kv4_func(**good)
        assert len(launches) == 1

    def test_varlen(self, launches):
        kc, vc = caches()
        table = torch.zeros(2, 1, dtype=torch.int32)
        for args in ((t(2, 1, 4, 64), kc, vc, i32(0, 1, 2), i32(0, 3), table), (t(2, 4, 64), kc, vc, i32(0, 2), i32(0, 3), table),
                     (t(2, 4, 64), kc, vc, None, i32(0, 3), table)):
            with pytest.raises(ValueError):
                mfa.flash_attn_varlen_kv4_func(*args)
        assert not launches

    def test_strides_reach_the_library(self, launches):
        kc, vc = caches(P=4, page=128, H=2, D=64)
        mfa.flash_attn_kv4_func(t(2, 3, 8, 64)[:, :, 2:6], kc, vc, i32(0, 3), torch.zeros(2, 5, dtype=torch.int32)[:, :3],
                                window_size=[7, -1], causal=True, softcap=2.0)
        p = launches[-1][1][0]
        c = p.cache
        assert (c.k.code_page_stride, c.k.code_row_stride, c.k.code_head_stride) == (2 * 128 * 32, 32, 128 * 32)
        assert (c.v.scale_page_stride, c.v.scale_row_stride, c.v.scale_head_stride) == (2 * 128 * 2, 2, 128 * 2)
        assert (c.max_pages, c.page_block_size, c.num_pages, c.block_table_batch_stride) == (3, 128, 4, 5)
        assert (p.q_batch_stride, p.q_seq_stride, p.q_head_stride) == (3 * 8 * 64, 8 * 64, 64)
        assert (p.window_left, p.window_right, p.causal, p.max_seqlen_k) == (7, -1, 1, 384)
        assert abs(p.scale - 0.125) < 1e-7 and p.softcap == 2.0


@pytest.mark.parametrize("pools,src,dst,exc", [
    ([t(4, 8), t(5, 8)], i32(0), i32(1), ValueError), ([t(4, 8)], i32(0, 1), i32(1), ValueError),
    ([t(4, 8)], [0], [1], ValueError), ([t(4, 8)], torch.zeros(1), i32(1), ValueError),
    ([t(4, 16)[:, ::2]], i32(0), i32(1), ValueError), ([t(1, 8).expand(4, 8)], i32(0), i32(1), ValueError),
    ([t(4, 1, 8).expand(4, 3, 8)], i32(0), i32(1), ValueError), ([None], i32(0), i32(1), ValueError),
    ([t(4, 8).requires_grad_()], i32(0), i32(1), NotImplementedError),
])
def test_copy_refusals(launches, pools, src, dst, exc):
    with pytest.raises(exc):
        mfa.copy_cache_pages(pools, src, dst)
    assert not launches


# --------------------------------------------------------------------------
# the C entry points


def refused(lib, rc, code, text):
    assert rc == code and text in lib.mfa_last_error().decode()


def fwd_params(D=64, H=4, Hkv=2):
    p = _hip.MfaKv4FwdParams()
    for pool in (p.cache.k, p.cache.v):
        pool.codes = pool.scales = 4096
        pool.code_page_stride, pool.code_row_stride, pool.code_head_stride = Hkv * 64 * D // 2, D // 2, 64 * D // 2
        pool.scale_page_stride, pool.scale_row_stride, pool.scale_head_stride = Hkv * 64 * D // 32, D // 32, 64 * D // 32
    p.cache.block_table = 4096
    p.cache.max_pages, p.cache.page_block_size, p.cache.num_pages = 4, 64, 8
    p.q = p.o = p.cache_seqlens = 4096
    p.q_batch_stride = p.o_batch_stride = H * D
    p.q_seq_stride = p.o_seq_stride = H * D
    p.q_head_stride = p.o_head_stride = D
    p.batch, p.seqlen_q, p.heads_q, p.heads_kv, p.head_dim = 2, 1, H, Hkv, D
    p.scale = 0.125
    p.window_left = p.window_right = -1
    p.dtype = _hip.MFA_DTYPE_BF16
    return p


@pytest.mark.parametrize("change,code,text", [
    (lambda p: setattr(p, "dtype", 2), -2, "dtype"), (lambda p: setattr(p, "head_dim", 80), -2, "head_dim"),
    (lambda p: setattr(p, "batch", -1), -1, "negative"), (lambda p: setattr(p, "heads_kv", 3), -1, "divide"),
    (lambda p: setattr(p, "softcap", float("nan")), -1, "softcap"), (lambda p: setattr(p, "window_left", -2), -1, "window"),
    (lambda p: setattr(p, "q", 4098), -1, "aligned"), (lambda p: setattr(p, "cache_seqlens", None), -1, "cache_seqlens"),
    (lambda p: setattr(p, "q_head_stride", 4), -1, "strides"), (lambda p: setattr(p, "seqlen_q", 1 << 30), -1, "too large"),
    (lambda p: setattr(p.cache, "page_block_size", 32), -1, "page_block_size"),
    (lambda p: setattr(p.cache, "block_table", None), -1, "block_table"),
    (lambda p: setattr(p.cache, "max_pages", 1 << 30), -1, "2^31"),
    (lambda p: setattr(p.cache.k, "codes", 4100), -1, "codes"), (lambda p: setattr(p.cache.v, "code_row_stride", 8), -1, "16 bytes"),
    (lambda p: setattr(p.cache.v, "scale_row_stride", -1), -1, ">= 0"),
    (lambda p: setattr(p.cache.k, "code_row_stride", 1 << 30), -1, "2 GiB"),
])
def test_c_attend(lib, change, code, text):
    p = fwd_params()
    assert lib.mfa_kv4_fwd_workspace_bytes(ctypes.byref(p)) > 0
    change(p)
    refused(lib, lib.mfa_kv4_fwd(ctypes.byref(p), None, 0, None), code, text)
    refused(lib, lib.mfa_kv4_fwd_workspace_bytes(ctypes.byref(p)), code, text)


def test_c_attend_workspace(lib):
    p = fwd_params()
    need = lib.mfa_kv4_fwd_workspace_bytes(ctypes.byref(p))
    refused(lib, lib.mfa_kv4_fwd(ctypes.byref(p), None, need, None), -1, "workspace")
    refused(lib, lib.mfa_kv4_fwd(ctypes.byref(p), 4096 + 16, need, None), -1, "aligned")
    refused(lib, lib.mfa_kv4_fwd(ctypes.byref(p), 4096, need - 1, None), -1, "needed")
    refused(lib, lib.mfa_kv4_fwd(None, None, 0, None), -1, "NULL")
    p.batch = 0
    assert lib.mfa_kv4_fwd(ctypes.byref(p), None, 0, None) == 0


def test_c_append(lib):
    def params():
        f = fwd_params()
        p = _hip.MfaKv4AppendParams()
        p.cache = f.cache
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
        refused(lib, lib.mfa_kv4_append(ctypes.byref(p), None), code, text)
    p = params()
    p.total = 0
    assert lib.mfa_kv4_append(ctypes.byref(p), None) == 0
    refused(lib, lib.mfa_kv4_append(None, None), -1, "NULL")


def test_c_copy_pages(lib):
    def params():
        p = _hip.MfaCopyPagesParams()
        p.pool[0] = (4096, 512, 256)
        p.src = p.dst = 4096
        p.pools, p.pairs, p.num_pages = 1, 3, 8
        return p
    for change, text in (
            (lambda p: setattr(p, "pools", 65), "pools"), (lambda p: setattr(p, "pairs", -1), "negative"),
            (lambda p: setattr(p, "src", None), "src"), (lambda p: setattr(p, "dst", 4097), "src"),
            (lambda p: setattr(p.pool[0], "page_stride", 128), "overlap"), (lambda p: setattr(p.pool[0], "base", None), "base"),
            (lambda p: setattr(p.pool[0], "page_bytes", -1), "page_bytes"),
            (lambda p: (setattr(p, "pairs", 1 << 30), setattr(p.pool[0], "page_bytes", 1 << 40), setattr(p.pool[0], "page_stride", 1 << 40)), "too large")):
        p = params()
        change(p)
        refused(lib, lib.mfa_copy_pages(ctypes.byref(p), None), -1, text)
    p = params()
    p.pairs = 0
    assert lib.mfa_copy_pages(ctypes.byref(p), None) == 0
    refused(lib, lib.mfa_copy_pages(None, None), -1, "NULL")


def test_c_norm_rope(lib):
    def params():
        b = _hip.MfaNormRopeBwdParams()
        p = b.fwd
        p.q = p.k = p.q_out = p.k_out = p.q_weight = p.k_weight = p.cos = p.sin = 4096
        p.q_seq_stride = p.k_seq_stride = 128
        p.q_head_stride = p.k_head_stride = 64
        p.batch, p.seqlen, p.heads_q, p.heads_kv, p.head_dim, p.rotary_dim, p.table_rows = 1, 5, 2, 2, 64, 64, 9
        p.dtype = p.dtype_weight = p.dtype_table = 1
        b.dq_out = b.dk_out = b.dq = b.dk = b.dq_weight = b.dk_weight = 4096
        return b
    assert lib.mfa_norm_rope_bwd_workspace_bytes(ctypes.byref(params())) > 0
    for change, code, text in (
            (dict(dtype=5), -1, "dtype"), (dict(dtype_weight=-1), -1, "dtype"), (dict(head_dim=129), -2, "head_dim"),
            (dict(head_dim=0), -2, "head_dim"), (dict(rotary_dim=3), -1, "rotary_dim"), (dict(rotary_dim=66), -1, "rotary_dim"),
            (dict(seqlen=-1), -1, "negative"), (dict(batch=1 << 20, seqlen=1 << 20), -1, "too large"), (dict(q=None), -1, "NULL"),
            (dict(k=4097), -1, "aligned"), (dict(cos=None), -1, "cos"), (dict(sin=4097), -1, "cos"),
            (dict(table_stride=-1), -1, "table_stride"), (dict(positions=4098), -1, "positions"),
            (dict(positions_batch_stride=-5), -1, "positions")):
        b = params()
        for k, v in change.items():
            setattr(b.fwd, k, v)
        refused(lib, lib.mfa_norm_rope(ctypes.byref(b.fwd), None), code, text)
        refused(lib, lib.mfa_norm_rope_bwd(ctypes.byref(b), 4096, 1 << 20, None), code, text)
    b = params()
    refused(lib, lib.mfa_norm_rope_bwd(ctypes.byref(b), None, 1 << 20, None), -1, "workspace")
    refused(lib, lib.mfa_norm_rope_bwd(ctypes.byref(b), 4096, 8, None), -1, "needed")
    b.dq_out = None
    refused(lib, lib.mfa_norm_rope_bwd(ctypes.byref(b), 4096, 1 << 20, None), -1, "NULL")
    b = params()
    b.fwd.batch = 0
    assert lib.mfa_norm_rope(ctypes.byref(b.fwd), None) == 0
    refused(lib, lib.mfa_norm_rope(None, None), -1, "NULL")


@pytest.mark.parametrize("field", ["q_weight", "k_weight"])
def test_c_norm_rope_weight_alignment(lib, field):
    p = _hip.MfaNormRopeParams()
    p.q = p.k = p.q_out = p.k_out = p.cos = p.sin = 4096
    p.q_seq_stride = p.k_seq_stride = p.q_head_stride = p.k_head_stride = 64
    p.batch, p.seqlen, p.heads_q, p.heads_kv, p.head_dim, p.rotary_dim, p.table_rows = 1, 1, 1, 1, 64, 64, 9
    p.dtype = p.dtype_weight = p.dtype_table = 1
    setattr(p, field, 4097)
    refused(lib, lib.mfa_norm_rope(ctypes.byref(p), None), -1, "weight")


def test_c_copy_pages_of_more_workgroups_than_a_launch_has(lib):
    p = _hip.MfaCopyPagesParams()
    p.pool[0] = (4097, 1 << 20, 1 << 20)  # (single bytes: at most 16 KB per workgroup)
    p.src = p.dst = 4096
    p.pools, p.pairs, p.num_pages = 1, 1 << 20, 8
    refused(lib, lib.mfa_copy_pages(ctypes.byref(p), None), -1, "too large")


def test_expanded_cache_cannot_be_written(launches):
    k = t(3, 2, 64)
    cu, lens, table = i32(0, 3), i32(0), i32(0, 1)[None]
    c = mfa.kv4_cache(2, 64, 2, 64, device="cpu")
    for which in (0, 1):
        e = tuple(x[:1].expand(2, -1, -1, -1) if i == which else x for i, x in enumerate(c))
        for caches in ((e, c), (c, e)):
            with pytest.raises(ValueError, match="expanded"):
                mfa.kv4_append(k, k, *caches, cu, lens, table)
    mfa.kv4_append(k, k, c, c, cu, lens, table)
    assert len(launches) == 1


def test_numbers_given_as_tensors_are_read_at_every_call(launches):
    """A tensor stands for its value, also after it was changed in place."""
    c = mfa.kv4_cache(2, 64, 2, 64, device="cpu")
    scale, eps = torch.tensor(0.5), torch.tensor(1e-3)
    q = t(1, 1, 2, 64)
    for i, (s, e) in enumerate(((0.5, 1e-3), (0.25, 1e-2))):
        scale.fill_(s)
        eps.fill_(e)
        mfa.flash_attn_kv4_func(q, c, c, i32(5), i32(0, 1)[None], softmax_scale=scale)
        mfa.qk_norm_rope(q, q, None, None, torch.zeros(9, 32), torch.zeros(9, 32), eps=eps)
        assert launches[2 * i][1][0].scale == s
        assert launches[2 * i + 1][1][0].eps == pytest.approx(e)


def test_forward_mode_derivatives_are_refused(launches):
    import torch.autograd.forward_ad as fw

    c = mfa.kv4_cache(2, 64, 2, 64, device="cpu")
    q, table = t(1, 3, 2, 64), i32(0, 1)[None]
    tables = torch.zeros(9, 32), torch.zeros(9, 32)
    with fw.dual_level():
        d = fw.make_dual(q, torch.ones_like(q))
        for call in (lambda: mfa.qk_norm_rope(d, q, None, None, *tables), lambda: mfa.qk_norm_rope(q, d, None, None, *tables),
                     lambda: mfa.flash_attn_kv4_func(d, c, c, i32(5), table),
                     lambda: mfa.kv4_append(d[0], q[0], c, c, i32(0, 3), i32(0), table)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        assert not launches
        mfa.qk_norm_rope(q, q, None, None, *tables)
    assert len(launches) == 1
