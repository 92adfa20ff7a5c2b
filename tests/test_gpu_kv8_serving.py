"""Steps of a server with the 8-bit cache: norm and rotation, append, attention, key weights
and eviction as one run, at once on several streams and in several threads, captured and
replayed in turn, beside forked sequences, and with the page checks on.  Runs of the same
step are compared for equal bits."""
from __future__ import annotations

import threading

import pytest
import torch

import mtlflashattn_amd as mfa
from kv8_util import DEV, bits, cu_of, i32

pytestmark = pytest.mark.gpu

CASES = [(1, 128, torch.bfloat16, 2), (2, 64, torch.float16, 2), (3, 96, torch.bfloat16, 20), (4, 32, torch.float16, 16)]


def serving_state(seed, D, dtype, Hkv):
    """Tensors of one server's step: a prompt chunk and decoding sequences."""
    g = torch.Generator().manual_seed(seed)
    Hq, page, lens, new = 4 * Hkv, 64, [0, 130, 700, 63], [100, 1, 1, 1]
    pages = sum(-(-(a + b) // page) for a, b in zip(lens, new)) + 2
    s = dict(kc=mfa.kv8_cache(pages, page, Hkv, D), vc=mfa.kv8_cache(pages, page, Hkv, D))
    for name in ("kc", "vc"):
        codes, scales = s[name]
        codes.view(torch.uint8).copy_(torch.randint(0, 120, codes.shape, generator=g, dtype=torch.uint8))
        scales.copy_(torch.randint(120, 124, scales.shape, generator=g, dtype=torch.uint8))
    ids, table = torch.randperm(pages, generator=g).tolist(), torch.full((4, 12), -1, dtype=torch.int32)
    for b, n in enumerate(zip(lens, new)):
        for i in range(-(-sum(n) // page)):
            table[b, i] = ids.pop()
    rows = lambda H: torch.randn(sum(new), H, D, generator=g).to(DEV, dtype)  # noqa: E731
    angle = torch.randn(900, D // 2, generator=g).to(DEV)
    pos = torch.cat([torch.arange(a, a + b) for a, b in zip(lens, new)]).to(DEV, torch.int32)
    s.update(q=rows(Hq), k=rows(Hkv), v=rows(Hkv), qw=torch.randn(D, generator=g).to(DEV, dtype), cos=angle.cos(), sin=angle.sin(),
             pos=pos, cu=cu_of(new), old=i32(*lens), total=i32(*(a + b for a, b in zip(lens, new))), table=table.to(DEV),
             w=torch.rand(pages, Hkv, page, generator=g).to(DEV).transpose(1, 2))
    s["start"] = [x.clone() for x in pools_of(s)]
    return s


def pools_of(s):
    return [*(c[0].view(torch.uint8) for c in (s["kc"], s["vc"])), s["kc"][1], s["vc"][1], s["w"]]


def serving_step(s):
    for x, start in zip(pools_of(s), s["start"]):
        x.copy_(start)
    q, k = mfa.qk_norm_rope(s["q"], s["k"], s["qw"], None, s["cos"], s["sin"], s["pos"])
    mfa.kv8_append(k, s["v"], s["kc"], s["vc"], s["cu"], s["old"], s["table"])
    out, lse = mfa.flash_attn_varlen_kv8_func(q, s["kc"], s["vc"], s["cu"], s["total"], s["table"], causal=True,
                                              return_softmax_lse=True)
    mfa.kv8_key_weights(q, s["kc"], lse, s["w"], s["total"], s["table"], s["cu"], causal=True)
    n = mfa.kv8_evict(s["kc"], s["vc"], s["w"], s["total"], s["table"], 90, 20)
    last = mfa.flash_attn_kv8_func(q[-4:, None], s["kc"], s["vc"], n, s["table"], causal=True)
    return [q, k, out, lse, n, last, *(x.clone() for x in pools_of(s))]


def same_bits(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_steps_on_several_streams_at_once():
    refs = [serving_step(serving_state(*c)) for c in CASES]
    assert all(bool(r[2].isfinite().all()) and bool(r[5].isfinite().all()) for r in refs)
    assert all(r[4].tolist() == [90, 90, 90, 64] for r in refs)
    states = [serving_state(*c) for c in CASES]
    streams = [torch.cuda.Stream() for _ in CASES]
    torch.cuda.synchronize()
    outs = [[] for _ in CASES]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[i].append(serving_step(states[i]))
    torch.cuda.synchronize()
    for ref, runs in zip(refs, outs):
        assert all(same_bits(got, ref) for got in runs)


def test_steps_in_several_threads_at_once():
    refs = [serving_step(serving_state(*c)) for c in CASES]
    states = [serving_state(*c) for c in CASES]
    torch.cuda.synchronize()
    outs, errors = [[] for _ in CASES], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    outs[i].append(serving_step(states[i]))
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # (shown by the main thread)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(CASES))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for ref, runs in zip(refs, outs):
        assert len(runs) == 5 and all(same_bits(got, ref) for got in runs)


def test_two_captured_steps_replayed_in_turn():
    """Two graphs with eager steps between the replays, inputs new every time."""
    states = [serving_state(*c) for c in CASES[1:3]]
    graphs, outs = [], []
    for s in states:
        serving_step(s)
    torch.cuda.synchronize()
    for s in states:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(serving_step(s))
        graphs.append(graph)
    for turn in range(4):
        for s in states:
            for name in ("q", "k", "v"):
                s[name].normal_()
        graphs[turn % 2].replay()
        graphs[1 - turn % 2].replay()
        torch.cuda.synchronize()
        got = [[t.clone() for t in o] for o in outs]
        for s, g in zip(states, got):
            ref = serving_step(s)
            torch.cuda.synchronize()
            assert same_bits(g, ref), turn


def test_forked_sequences():
    """A fork shares its full pages and copies the last one: the bits of two sequences of their own."""
    D, Hkv, Hq, page, n = 64, 2, 8, 64, 150
    g = torch.Generator().manual_seed(5)
    rows = lambda m, H: torch.randn(m, H, D, generator=g).to(DEV, torch.bfloat16)  # noqa: E731
    k, v = rows(n, Hkv), rows(n, Hkv)
    k2, v2, q = rows(2, Hkv), rows(2, Hkv), rows(2, Hq)
    runs = []
    for forked in (False, True):
        kc, vc = mfa.kv8_cache(8, page, Hkv, D), mfa.kv8_cache(8, page, Hkv, D)
        if forked:
            mfa.kv8_append(k, v, kc, vc, cu_of([n]), i32(0), i32(0, 1, 2)[None])
            mfa.copy_cache_pages([kc[0], kc[1], vc[0], vc[1]], i32(2), i32(5))
            table = i32(0, 1, 2, 0, 1, 5).view(2, 3)
        else:
            table = i32(0, 1, 2, 3, 4, 5).view(2, 3)
            mfa.kv8_append(torch.cat((k, k)), torch.cat((v, v)), kc, vc, cu_of([n, n]), i32(0, 0), table)
        mfa.kv8_append(k2, v2, kc, vc, cu_of([1, 1]), i32(n, n), table)
        runs.append([mfa.flash_attn_kv8_func(q[:, None], kc, vc, i32(n + 1, n + 1), table, causal=True),
                     *(x[2] for x in (*bits(kc), *bits(vc))), *(x[5] for x in (*bits(kc), *bits(vc)))])
    assert same_bits(*runs)


def test_page_checks_on_request(monkeypatch):
    monkeypatch.setenv("MTLFLASHATTN_CHECK_PAGES", "1")
    kc, vc = mfa.kv8_cache(3, 64, 2, 64), mfa.kv8_cache(3, 64, 2, 64)
    w = torch.zeros(3, 64, 2, device=DEV)
    q, lse = torch.randn(1, 1, 2, 64, device=DEV, dtype=torch.bfloat16), torch.zeros(1, 2, 1, device=DEV)
    k = torch.randn(3, 2, 64, device=DEV)
    good, bad = i32(2, 9)[None], i32(5, 1)[None]
    mfa.flash_attn_kv8_func(q, kc, vc, i32(60), good)
    mfa.kv8_append(k, k, kc, vc, i32(0, 3), i32(61), good)
    mfa.kv8_key_weights(q, kc, lse, w, i32(64), good)
    mfa.kv8_evict(kc, vc, w, i32(64), good, 10, 5)
    mfa.kv8_evict(kc, vc, w, i32(65), good, 10, 5, max_seqlen_k=64)
    for call in (lambda: mfa.flash_attn_kv8_func(q, kc, vc, i32(65), good),
                 lambda: mfa.flash_attn_kv8_func(q, kc, vc, i32(5), bad),
                 lambda: mfa.kv8_append(k, k, kc, vc, i32(0, 3), i32(62), good),
                 lambda: mfa.kv8_append(k, k, kc, vc, i32(0, 3), i32(126), good),
                 lambda: mfa.kv8_key_weights(q, kc, lse, w, i32(65), good),
                 lambda: mfa.kv8_evict(kc, vc, w, i32(65), good, 10, 5),
                 lambda: mfa.kv8_evict(kc, vc, w, i32(5), bad, 10, 5)):
        with pytest.raises(ValueError):
            call()
