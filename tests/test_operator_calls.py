"""Calls of the operators around the attention call that their first tests leave out,
on the CPU: the device predicate patched and the launches recorded instead of made."""
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


@pytest.fixture
def launches(monkeypatch):
    """(name, parameters) of every launch; CPU tensors count as ROCm tensors."""
    calls = []
    monkeypatch.setattr(_kernel, "_is_rocm_tensor", lambda x: True)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 0, raising=False)
    for name in ("norm_rope", "norm_rope_bwd", "kv4_append", "kv4_fwd", "copy_pages"):
        monkeypatch.setattr(_hip, name, lambda *a, name=name: calls.append((name, a[0])))
    for name in ("kv4_fwd_workspace_bytes", "norm_rope_bwd_workspace_bytes"):
        monkeypatch.setattr(_hip, name, lambda p: 0)
    return calls


class TestSavedTensorHooks:
    """The backward of qk_norm_rope reads what the hooks give back, by its own strides."""

    def call(self, unpack):
        """Gradients of views of packed tensors, whose saved copies `unpack` gives back."""
        qkv = t(5, 12, 64).requires_grad_()
        w = t(2, 64)
        table = t(9, 96, dtype=torch.float32)
        pos = torch.zeros(5, 2, dtype=torch.int64)
        with torch.autograd.graph.saved_tensors_hooks(lambda x: x, unpack):
            q, k = mfa.qk_norm_rope(qkv[:, :4], qkv[:, 4:8], w[0], w[1], table[:, :32], table[:, 32:64], pos[:, 0])
        torch.autograd.grad((q, k), qkv, (torch.ones_like(q), torch.ones_like(k)))

    def test_dense_copies(self, launches):
        given = []

        def dense(x):
            given.append(x.contiguous().clone())
            return given[-1]

        self.call(dense)
        (_, fwd), (_, bwd) = launches
        assert (fwd.q_seq_stride, fwd.k_seq_stride, fwd.table_stride) == (12 * 64, 12 * 64, 96)
        b = bwd.fwd
        assert (b.q_seq_stride, b.q_head_stride, b.k_seq_stride, b.k_head_stride) == (4 * 64, 64, 4 * 64, 64)
        assert b.table_stride == 32
        assert [b.q, b.k, b.q_weight, b.k_weight, b.cos, b.sin, b.positions] == [x.data_ptr() for x in given]

    def test_rows_that_are_not_contiguous(self, launches):
        """A copy with other strides, which the kernel cannot address, is made dense first."""
        self.call(lambda x: x.transpose(0, -1).clone(memory_format=torch.contiguous_format).transpose(0, -1)
                  if x.dim() == 3 else x)
        b = launches[1][1].fwd
        assert (b.q_seq_stride, b.q_head_stride, b.k_seq_stride, b.k_head_stride) == (4 * 64, 64, 4 * 64, 64)
        assert b.table_stride == 96

    @pytest.mark.parametrize("unpack", [lambda x: x[:3], lambda x: x[..., :2, :] if x.dim() == 3 else x,
                                        lambda x: x.double() if x.dim() == 3 else x])
    def test_other_sizes_or_types_are_refused(self, launches, unpack):
        with pytest.raises((ValueError, NotImplementedError), match="mtlflashattn_amd"):
            self.call(unpack)
        assert len(launches) == 1

    def test_without_hooks(self, launches):
        qkv = t(5, 12, 64).requires_grad_()
        q, k = mfa.qk_norm_rope(qkv[:, :4], qkv[:, 4:8], None, None, t(9, 32), t(9, 32))
        torch.autograd.grad((q, k), qkv, (torch.ones_like(q), torch.ones_like(k)))
        b = launches[1][1].fwd
        assert (b.q_seq_stride, b.k_seq_stride) == (12 * 64, 12 * 64)


@pytest.mark.parametrize("table", [t(9000, 0), t(9000, 64)[:, :0]])
def test_tables_without_columns_have_one_row(launches, table):
    mfa.qk_norm_rope(t(5, 4, 64), t(5, 2, 64), None, None, table, table)
    p = launches[0][1]
    assert (p.rotary_dim, p.table_rows, p.table_stride) == (0, 9000, 0)


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_build.LIB_PATH):
        _build.build()
    return _hip.load()


def test_no_sequences_need_no_table(lib):
    """A table of no rows has no memory: torch gives a null pointer for it."""
    f = _hip.MfaKv4FwdParams()
    c = f.cache
    for pool in (c.k, c.v):
        pool.codes = pool.scales = 4096
        pool.code_page_stride, pool.code_row_stride, pool.code_head_stride = 64 * 32, 32, 64 * 32
        pool.scale_page_stride, pool.scale_row_stride, pool.scale_head_stride = 64 * 2, 2, 64 * 2
    c.max_pages, c.page_block_size, c.num_pages = 4, 64, 8
    f.q = f.o = 4096
    f.q_seq_stride = f.o_seq_stride = f.q_head_stride = f.o_head_stride = 64
    f.seqlen_q, f.heads_q, f.heads_kv, f.head_dim, f.scale, f.dtype = 1, 1, 1, 64, 0.125, _hip.MFA_DTYPE_BF16
    f.window_left = f.window_right = -1
    a = _hip.MfaKv4AppendParams()
    a.cache, a.k, a.v, a.cu_seqlens = c, 4096, 4096, 4096
    a.heads_kv, a.head_dim, a.dtype = 1, 64, _hip.MFA_DTYPE_BF16
    assert lib.mfa_kv4_fwd(ctypes.byref(f), None, 0, None) == 0
    assert lib.mfa_kv4_append(ctypes.byref(a), None) == 0
    f.batch = f.total_q = a.batch = a.total = 1
    f.cache_seqlens = a.cache_seqlens = 4096
    assert lib.mfa_kv4_fwd(ctypes.byref(f), None, 0, None) == -1 and b"block_table" in lib.mfa_last_error()
    assert lib.mfa_kv4_append(ctypes.byref(a), None) == -1 and b"block_table" in lib.mfa_last_error()


class TestVersionCounters:
    """A graph that saved a pool notices that the pool was written."""

    def saved(self, pool):
        x = torch.ones(pool.shape, requires_grad=True)
        return (x * pool).sum()  # saves the pool

    def test_copied_pages(self, launches):
        pools = [torch.zeros(4, 8), torch.zeros(4, 3, 8)[:, 1]]
        losses = [self.saved(p) for p in pools]
        mfa.copy_cache_pages(pools, i32(0), i32(1))
        for loss in losses:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                loss.backward()

    def test_appended_rows(self, launches):
        kc, vc = (mfa.kv4_cache(2, 64, 2, 64, device="cpu") for _ in range(2))
        losses = [self.saved(p) for p in (*kc, *vc)]
        mfa.kv4_append(t(3, 2, 64), t(3, 2, 64), kc, vc, i32(0, 3), i32(0), i32(0, 1)[None])
        for loss in losses:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                loss.backward()

    def test_inference_tensors(self, launches):
        with torch.inference_mode():
            pool = torch.zeros(4, 8)
            kc, vc = (mfa.kv4_cache(2, 64, 2, 64, device="cpu") for _ in range(2))
        for mode in (True, False):
            with torch.inference_mode(mode):
                mfa.copy_cache_pages([pool], i32(0), i32(1))
                mfa.kv4_append(t(3, 2, 64), t(3, 2, 64), kc, vc, i32(0, 3), i32(0), i32(0, 1)[None])
        assert len(launches) == 4

    def test_read_only_calls(self, launches):
        c = mfa.kv4_cache(2, 64, 2, 64, device="cpu")
        before = [x._version for x in c]
        mfa.flash_attn_kv4_func(t(1, 1, 2, 64), c, c, i32(3), i32(0, 1)[None])
        assert [x._version for x in c] == before


class TestSizesBeyond32Bits:
    """Sizes that the library's 32-bit fields cannot hold are refused, not cut off."""

    @pytest.mark.parametrize("n", [1 << 31, (1 << 32) + 3])
    def test_append(self, launches, n):
        c = mfa.kv4_cache(2, 64, 2, 64, device="cpu")
        k = t(1, 2, 64).expand(n, 2, 64)
        with pytest.raises(ValueError, match="2\\^31"):
            mfa.kv4_append(k, k, c, c, i32(0, 3), i32(0), i32(0, 1)[None])
        assert not launches

    @pytest.mark.parametrize("n", [1 << 31, (1 << 32) + 3])
    def test_pages(self, launches, n):
        c = tuple(x[:1].expand(n, -1, -1, -1) for x in mfa.kv4_cache(2, 64, 2, 64, device="cpu"))
        with pytest.raises(ValueError, match="2\\^31"):
            mfa.flash_attn_kv4_func(t(1, 1, 2, 64), c, c, i32(3), i32(0, 1)[None])
        with pytest.raises(ValueError, match="2\\^31"):
            mfa.copy_cache_pages([torch.empty(n, 0)], i32(0), i32(1))
        with pytest.raises(ValueError, match="2\\^31"):
            mfa.copy_cache_pages([t(4, 8)], i32(0).expand(n), i32(1).expand(n))
        assert not launches

    @pytest.mark.parametrize("cols", [1 << 25, (1 << 26), (1 << 26) + 1])
    def test_tables(self, launches, cols):
        """Tables that name 2^31 rows and more (the memory is not touched)."""
        c = mfa.kv4_cache(2, 64, 2, 64, device="cpu")
        table = torch.empty(1, cols, dtype=torch.int32)
        with pytest.raises(ValueError, match="2\\^31"):
            mfa.flash_attn_kv4_func(t(1, 1, 2, 64), c, c, i32(3), table)
        with pytest.raises(ValueError, match="2\\^31"):
            mfa.kv4_append(t(3, 2, 64), t(3, 2, 64), c, c, i32(0, 3), i32(0), table)
        assert not launches

    @pytest.mark.parametrize("n", [1 << 31, (1 << 32) + 3])
    def test_norm_and_rotation(self, launches, n):
        table, few = t(1, 4).expand(n, 4), t(1, 4)
        x = t(5, 2, 64)
        with pytest.raises(ValueError, match="2\\^31"):
            mfa.qk_norm_rope(x, x, None, None, table, table)
        q = t(1, 1, 64).expand(n, 1, 64)
        with pytest.raises(ValueError, match="2\\^31"):
            mfa.qk_norm_rope(q, q, None, None, few, few)
        assert not launches

    @pytest.mark.parametrize("window", [(1 << 31, 1 << 32), (1 << 40, 1 << 63)])
    def test_windows_are_unbounded(self, launches, window):
        c = mfa.kv4_cache(2, 64, 2, 64, device="cpu")
        mfa.flash_attn_kv4_func(t(1, 1, 2, 64), c, c, i32(3), i32(0, 1)[None], window_size=window)
        p = launches[0][1]
        assert min(p.window_left, p.window_right) >= (1 << 31) - 1
