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
    assert _hip.kv4_fwd_workspace_bytes(p) == 0
    _hip.kv4_fwd(p, None, 0, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert not out.any() and bool((lse == float("-inf")).all())


LEVELS = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("lq,Hq,window", [(1, 4, (40, 0)), (5, 4, (-1, 0)), (9, 6, (33, 0)), (70, 4, (-1, 0)),
                                          (70, 4, (50, 3)), (150, 2, (-1, -1))])
def test_values_beyond_the_range_reach_only_the_rows_that_see_them(lq, Hq, window, D, dtype):
    """Groups of V with elements of 2^128 and more (scales 2^126 and 2^127, what
    kv4_append makes of the type's largest values): every row that masks their key
    has the bits that it has without them; bf16 rows that see one get it as +/-1.5 *
    2^127.  One such group per head and 32 elements, so a row's sum stays below 2^128;
    bound there: the rounding of the result, and of its probability to one bf16 term
    (2^-8 each of the largest value), next to 3e-4 for the rest."""
    L, page, pages = 333, 64, 9
    g = torch.Generator().manual_seed(D)
    kc, vc = (tuple(torch.randint(lo, hi, (pages, 2, page, n), generator=g, dtype=torch.uint8).to(DEV).transpose(1, 2)
                    for n, lo, hi in ((D // 2, 0, 256), (D // 32, 123, 127))) for _ in range(2))
    table = torch.randperm(pages, generator=g)[None].to(DEV, torch.int32)
    q, lens = torch.randn(1, lq, Hq, D, generator=g).to(DEV, dtype), i32(L)

    def call():
        return mfa.flash_attn_kv4_func(q, kc, vc, lens, table, window_size=window)[0].cpu()

    i, j = torch.arange(lq)[:, None] + L - lq, torch.arange(L)[None]
    seen = torch.ones(lq, L, dtype=torch.bool)
    if window[0] >= 0:
        seen &= j >= i - window[0]
    if window[1] >= 0:
        seen &= j <= i + window[1]
    groups = D // 32
    spots = {(0, 0): (L - 1, 253), (1, groups - 1): (L - lq // 2 - 1, 254)}
    spots.setdefault((0, groups - 1), (max(L - lq - 36, 0), 254))
    spots.setdefault((1, 0), (258, 253))
    want = torch.zeros(lq, Hq, D, dtype=torch.bool)
    for (h, grp), (key, byte) in spots.items():
        p = table[0, key // page].item()
        vc[0][p, key % page, h, 16 * grp:16 * grp + 8] = torch.tensor([0x67, 0xEF, 0x54, 0xDC, 0x32, 0xBA, 0x10, 0x98],
                                                                      dtype=torch.uint8, device=DEV)
    clean = call()  # (the codes with ordinary scales)
    for (h, grp), (key, byte) in spots.items():
        vc[1][table[0, key // page].item(), key % page, h, grp] = byte
        want[:, h * Hq // 2:(h + 1) * Hq // 2, 32 * grp:32 * grp + 32] |= seen[:, key][:, None, None]
    out = call()
    assert torch.equal(out[~want], clean[~want])
    if dtype == torch.float16:
        return
    rows = []
    for codes, scales in (kc, vc):
        codes, scales = (x.cpu()[table[0].cpu().long()].flatten(0, 1)[:L] for x in (codes, scales))
        x = torch.stack((LEVELS[codes.long() & 15], LEVELS[codes.long() >> 4]), -1).flatten(-2)
        x = x * torch.pow(2.0, scales.double() - 127).repeat_interleave(32, -1)
        rows.append(x.clamp(-1.5 * 2.0 ** 127, 1.5 * 2.0 ** 127))
    ref = torch.zeros(lq, Hq, D, dtype=torch.float64)
    for h in range(Hq):
        s = (q[0, :, h].cpu().double() @ rows[0][:, h * 2 // Hq].T / D ** 0.5).masked_fill(~seen, -float("inf"))
        p = torch.softmax(s, -1)
        ref[:, h] = p @ rows[1][:, h * 2 // Hq]
    err = (out.double() - ref).abs()[want]
    assert bool((err <= (2.0 ** -8 * 2 + 3e-4) * 1.5 * 2.0 ** 127).all()) and bool(out[want].isfinite().all())


@pytest.mark.parametrize("lq,Hq,window", [(1, 4, (100, 300)), (5, 4, (0, 300)), (70, 4, (100, 300)),
                                          (70, 4, (100, 1 << 29)), (3, 4, (100, 1 << 29)), (70, 4, (100, -1)), (3, 4, (100, -1))])
def test_right_window_at_the_longest_sequence(lq, Hq, window):
    """The last positions of 2^31 - 256 keys (a table that repeats five pages), whose
    right window's end has no 32-bit number, nor the chunks of the window that lie
    behind the last key: the bits of the same keys in a short
    sequence with a window that ends behind them."""
    page, pages, D, cols = 256, 5, 64, (1 << 23) - 1
    g = torch.Generator().manual_seed(lq)
    kc, vc = (tuple(torch.randint(lo, hi, (pages, 2, page, n), generator=g, dtype=torch.uint8).to(DEV).transpose(1, 2)
                    for n, lo, hi in ((D // 2, 0, 256), (D // 32, 123, 127))) for _ in range(2))
    q = torch.randn(1, lq, Hq, D, generator=g).to(DEV, torch.bfloat16)
    table = (torch.arange(cols, dtype=torch.int32, device=DEV) % pages)[None]
    first = (cols - 4) // 2 * 2  # (the last pages from a multiple of a chunk of both)
    short = table[:, first:].contiguous()
    want = mfa.flash_attn_kv4_func(q, kc, vc, i32(short.shape[1] * page), short, window_size=(window[0], 300))
    got = mfa.flash_attn_kv4_func(q, kc, vc, i32(cols * page), table, window_size=window)
    assert bool(want.any(-1).all()) and torch.equal(got, want)


@pytest.mark.parametrize("lq", [1, 40])
def test_left_windows_above_2_30_keys(lq):
    """2^31 - 256 keys that repeat every 1280: a window of w keys has w / 1280 of their
    sum, so the log-sum-exp differs from the whole row's by the logarithm of the shares
    (a walk adds at most 2^31 / (512 * 64) = 2^16 blocks in fp32: 2^16 * 2^-24 = 2^-8 of
    either sum)."""
    page, pages, D, cols = 256, 5, 32, (1 << 23) - 1
    g = torch.Generator().manual_seed(lq)
    kc, vc = (tuple(torch.randint(lo, hi, (pages, 1, page, n), generator=g, dtype=torch.uint8).to(DEV).transpose(1, 2)
                    for n, lo, hi in ((D // 2, 0, 256), (D // 32, 123, 127))) for _ in range(2))
    q = torch.randn(1, lq, 2, D, generator=g).to(DEV, torch.bfloat16)
    table = (torch.arange(cols, dtype=torch.int32, device=DEV) % pages)[None]
    n = cols * page

    def lse(left):
        return mfa.flash_attn_kv4_func(q, kc, vc, i32(n), table, causal=True, window_size=(left, 0),
                                       return_softmax_lse=True)[1]

    whole = lse(-1)
    assert torch.equal(lse(n), whole) and torch.equal(lse((1 << 31) - 1), whole) and torch.equal(lse(1 << 40), whole)
    for w in (5 << 28, 3 << 28):
        want = whole.double() + torch.log(torch.tensor(w / n, dtype=torch.float64))
        assert float((lse(w).double() - want).abs().max()) <= 2.0 ** -8 * 2


def test_gradients_of_a_checkpointed_block():
    """Recomputed inputs (torch.utils.checkpoint works through saved-tensor hooks)."""
    from torch.utils.checkpoint import checkpoint

    qkv = torch.randn(200, 12, 64, device=DEV, dtype=torch.bfloat16).requires_grad_()
    w = torch.ones(64, device=DEV, dtype=torch.bfloat16).requires_grad_()
    table = torch.randn(200, 32, device=DEV)

    def block(x):
        q, k = mfa.qk_norm_rope(x[:, :8], x[:, 8:10], w, w, table, table)
        return mfa.flash_attn_func(q[None], k[None], x[None, :, 10:], causal=True)

    up = torch.randn(1, 200, 8, 64, device=DEV, dtype=torch.bfloat16)
    want = torch.autograd.grad(block(qkv), (qkv, w), up)
    got = torch.autograd.grad(checkpoint(block, qkv, use_reentrant=False), (qkv, w), up)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
