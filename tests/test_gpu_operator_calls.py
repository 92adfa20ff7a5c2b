"""Calls of the operators around the attention call that their first tests leave out."""
from __future__ import annotations

import pytest
import torch

import mtlflashattn_amd as mfa

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("how", ["cpu", "dense"])
def test_gradients_through_saved_tensor_hooks(how, dtype):
    """Hooks that give back dense copies of views: the bits of the call without hooks
    (the same values, sizes and alignment, so the same sums in the same order)."""
    g = torch.Generator().manual_seed(1)
    Hq, Hkv, D, L = 8, 2, 64, 300
    qkv = torch.randn(L, Hq + 2 * Hkv, D, generator=g).to(DEV, dtype).requires_grad_()
    w = [(1 + 0.2 * torch.randn(D, generator=g)).to(DEV, dtype).requires_grad_() for _ in range(2)]
    table = torch.randn(4096, 3 * D, generator=g).to(DEV)
    cos, sin = table[:, :D // 2], table[:, D // 2:D]
    pos = torch.randint(0, 4096, (L, 2), generator=g).to(DEV)[:, 0]
    ups = [torch.randn(L, h, D, generator=g).to(DEV, dtype) for h in (Hq, Hkv)]

    def grads():
        outs = mfa.qk_norm_rope(qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], *w, cos, sin, pos)
        return torch.autograd.grad(outs, (qkv, *w), ups)

    want = grads()
    with (torch.autograd.graph.save_on_cpu() if how == "cpu" else
          torch.autograd.graph.saved_tensors_hooks(lambda x: x.contiguous().clone(), lambda x: x)):
        got = grads()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D", [64, 36])
@pytest.mark.parametrize("wide", [0, 64])
def test_norm_without_rotation(wide, D, interleaved):
    """Tables of no columns and many rows (empty, or a slice of wide ones): the norm
    alone, forward and backward, at every position.  Bounds as in
    test_gpu_norm_rope: an output 32, a gradient 64 steps of 2^-24 of the row's largest."""
    g = torch.Generator().manual_seed(2)
    rows = 65536
    table = torch.randn(rows, wide, generator=g).to(DEV)[:, :0]
    pos = torch.cat((torch.arange(rows - 40, rows), torch.randint(0, rows, (60,), generator=g))).to(DEV)
    x = torch.randn(100, 3, D, generator=g).to(DEV).requires_grad_()
    up = torch.randn(100, 3, D, generator=g).to(DEV)
    out, _ = mfa.qk_norm_rope(x, x.detach(), None, None, table, table, pos, interleaved=interleaved)
    dx, = torch.autograd.grad(out, x, up)
    y = x.detach().double().cpu().requires_grad_()
    ref = y / torch.sqrt(y.square().mean(-1, keepdim=True) + 1e-6)
    dref, = torch.autograd.grad(ref, y, up.double().cpu())
    for got, want, steps in ((out.detach(), ref.detach(), 32), (dx, dref, 64)):
        err = (got.double().cpu() - want).abs()
        scale = want.abs().amax(-1, keepdim=True)
        if steps == 64:  # rs max|h|
            rs = 1 / torch.sqrt(y.detach().square().mean(-1, keepdim=True) + 1e-6)
            scale = scale + rs * up.double().cpu().abs().amax(-1, keepdim=True)
        assert bool((err <= steps * 2.0 ** -24 * scale).all())
    fwd, _ = mfa.qk_norm_rope(x.detach(), x.detach(), None, None, table, table, interleaved=interleaved)
    assert torch.equal(fwd, out.detach())


def test_calls_of_no_sequences():
    """A step without sequences: nothing to write, rows of no sequence are 0 and -inf."""
    kc, vc = (mfa.kv4_cache(3, 64, 2, 64) for _ in range(2))
    cu, none = i32(0), torch.zeros(0, dtype=torch.int32, device=DEV)
    for table in (torch.zeros(0, 4, dtype=torch.int32, device=DEV), torch.zeros(0, 0, dtype=torch.int32, device=DEV)):
        q = torch.randn(0, 2, 4, 64, device=DEV, dtype=torch.bfloat16)
        out, lse = mfa.flash_attn_kv4_func(q, kc, vc, none, table, return_softmax_lse=True)
        assert out.shape == q.shape and lse.shape == (0, 4, 2)
        q = torch.randn(5, 4, 64, device=DEV, dtype=torch.bfloat16)
        out, lse = mfa.flash_attn_varlen_kv4_func(q, kc, vc, cu, none, table, return_softmax_lse=True)
        assert not out.any() and bool((lse == float("-inf")).all()) and lse.shape == (4, 5)
        assert mfa.kv4_append(q[:0, :2], q[:0, :2], kc, vc, cu, none, table) is None
        assert mfa.kv4_append(q[:, :2], q[:, :2], kc, vc, cu, none, table) is None
        assert not any(t.any() for t in (*kc, *vc))


def test_values_of_tokens_of_no_sequence():
    """What the cache would hold for them, also where there is no sequence at all."""
    k, v = (torch.randn(300, 2, 64, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    pools = [mfa.kv4_cache(8, 64, 2, 64) for _ in range(2)]
    table, none = i32(*range(8))[None], torch.zeros(0, dtype=torch.int32, device=DEV)
    want = mfa.kv4_append(k, v, *pools, i32(0, 300), i32(0), table, return_values=True)
    held = [t.clone() for c in pools for t in c]
    marks = [torch.full_like(k, 7.0) for _ in range(4)]  # (memory that the results may come to lie in)
    del marks
    some = mfa.kv4_append(k, v, *pools, i32(0, 0), i32(0), table, return_values=True)
    got = mfa.kv4_append(k, v, *pools, i32(0), none, table[:0], return_values=True)
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, some, got))
    assert all(torch.equal(a, b) for a, b in zip(held, (t for c in pools for t in c)))


def test_c_rows_of_no_sequences_are_cleared():
    """mfa_kv4_fwd with rows but no sequences, through the C parameters."""
    from mtlflashattn_amd import _hip

    out = torch.full((40, 8, 64), 7.0, device=DEV, dtype=torch.bfloat16)
    lse = torch.full((8, 40), 7.0, device=DEV)
    cu, codes, scales = i32(0), torch.zeros(2, 2, 64, 32, dtype=torch.uint8, device=DEV), torch.zeros(2, 2, 64, 2, dtype=torch.uint8, device=DEV)
    p = _hip.MfaKv4FwdParams()
    for pool in (p.cache.k, p.cache.v):
        pool.codes, pool.scales = codes.data_ptr(), scales.data_ptr()
        pool.code_page_stride, pool.code_row_stride, pool.code_head_stride = codes.stride(0), codes.stride(2), codes.stride(1)
        pool.scale_page_stride, pool.scale_row_stride, pool.scale_head_stride = scales.stride(0), scales.stride(2), scales.stride(1)
    p.cache.max_pages, p.cache.page_block_size, p.cache.num_pages = 4, 64, 2
    p.q = p.o = out.data_ptr()
    p.q_seq_stride = p.o_seq_stride = 8 * 64
    p.q_head_stride = p.o_head_stride = 64
    p.softmax_lse, p.lse_head_stride, p.cu_seqlens_q = lse.data_ptr(), 40, cu.data_ptr()
    p.total_q, p.heads_q, p.heads_kv, p.head_dim, p.scale = 40, 8, 2, 64, 0.125
    p.window_left = p.window_right = -1
    p.dtype = _hip.MFA_DTYPE_BF16
    n = _hip.kv4_fwd_workspace_bytes(p)
    ws = torch.empty(max(n, 1), dtype=torch.uint8, device=DEV)
    _hip.kv4_fwd(p, ws.data_ptr(), n, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert not out.any() and bool((lse == float("-inf")).all())
