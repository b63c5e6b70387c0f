"""Attention over the 8-bit cache for batches of more sequences than a wave has lanes,
rows of more records than that, and calls that run beside others; within the bound of
kv8_reference.attention, as in test_gpu_kv8_attention."""
import numpy as np
import pytest
import torch

import kv8_reference as ref
from test_gpu_kv8_attention import (DEV, cache, check_decode, check_prefill, decode, dev,
                                    on_device, queries)

pytestmark = pytest.mark.gpu


def batch_lens(r, B, most):
    """Short contexts, empty ones and a few long ones, the last lane's and the next
    wave's first among them."""
    lens = r.integers(0, 90, B)
    lens[r.random(B) < 0.15] = 0
    for b in (0, 63, 64, B - 1):
        lens[b] = r.integers(most // 2, most)
    return [int(n) for n in lens]


@pytest.mark.parametrize("d,H,G,code", [(64, 1, 2, "fp8"), (128, 2, 4, "int8"), (256, 1, 3, "fp8")])
@pytest.mark.parametrize("B", [65, 130, 200])
def test_decode_of_many_sequences(tq4, B, d, H, G, code):
    r = np.random.default_rng(B + d)
    lens = batch_lens(r, B, 700)
    c = cache(r, lens, H, 16, d, code)
    q = queries(r, B, H * G, d, "bf16", 2.0)
    check_decode(tq4, q, c, lens, code)
    check_decode(tq4, q, c, lens, code, num_splits=3)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d,G", [(64, 1), (128, 2), (256, 3)])
@pytest.mark.parametrize("B,most", [(65, 3), (130, 5), (70, 60), (140, 50)])
def test_prefill_of_many_sequences(tq4, B, most, d, G, causal):
    """Few rows a sequence, and row tiles of the prompt's kernel; sequences without
    rows between."""
    r = np.random.default_rng(B + d + most)
    rows = r.integers(0, most + 1, B)
    rows[r.random(B) < 0.2] = 0
    rows[63], rows[64], rows[B - 1] = most, most, 1
    lens = [max(a, int(b)) for a, b in zip(batch_lens(r, B, 500), rows)]
    c = cache(r, lens, 1, 16, d, "fp8")
    q = queries(r, int(rows.sum()) + 2, G, d, "bf16", 2.0)
    check_prefill(tq4, q, c, lens, [int(n) for n in rows], "fp8", causal)


@pytest.mark.parametrize("K", [65, 128, 256])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_decode_of_many_records(tq4, d, K):
    """Up to 141 records a row, more than a wave reads at once."""
    r = np.random.default_rng(d + K)
    lens = [4200, 9000, 70]
    c = cache(r, lens, 1, 16, d, "int8")
    # scores that grow and fall along the context: the maximum is in either half
    for b, n in enumerate(lens):
        pages = c[3][b][c[3][b] >= 0]
        c[2][0, pages, 0] = 2.0 ** (-9 + 3 * np.sin(np.linspace(0, 5 + b, len(pages))))
    check_decode(tq4, queries(r, 3, 4, d, "bf16"), c, lens, "int8", num_splits=K)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_streamed_decode_of_many_records(tq4, d):
    """Two long sequences in shares: 79 records a row."""
    r = np.random.default_rng(d)
    lens = [20000, 19333]
    kc, vc, sc, tables = cache(r, lens, 1, 16, d, "fp8")
    far = np.full((2, 450000 // 16), -1, np.int32)
    far[:, :tables.shape[1]] = tables
    q = queries(r, 2, 3, d, "bf16")
    check_decode(tq4, q, (kc, vc, sc, far), lens, "fp8", num_splits=0)
    check_prefill(tq4, queries(r, 4, 3, d, "bf16"), (kc, vc, sc, far), lens, [3, 1], "fp8", True)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_rows_with_splits_do_not_depend_on_the_batch(tq4, d):
    """With num_splits a row's bits are its own sequence's: alone, in a batch, in
    another order of it. (The tables have one width: the parts are of a sequence's
    tokens, not of its table's.)"""
    r = np.random.default_rng(d)
    B = 70
    lens = batch_lens(r, B, 900)
    c = cache(r, lens, 2, 16, d, "fp8")
    q = queries(r, B, 8, d, "bf16")
    order = r.permutation(B)
    for K in (1, 3, 40):
        whole = decode(tq4, q, c, lens, "fp8", num_splits=K)
        mixed = decode(tq4, q[order], (*c[:3], c[3][order]), [lens[b] for b in order], "fp8",
                       num_splits=K)
        assert torch.equal(mixed, whole[torch.from_numpy(order).to(DEV)])
        for b in (0, 63, 64, B - 1):
            one = decode(tq4, q[b:b + 1], (*c[:3], c[3][b:b + 1]), lens[b:b + 1], "fp8",
                         num_splits=K)
            assert torch.equal(one[0], whole[b])


def different_calls(tq4, n):
    """n decodes and n prefills over one cache that differ in everything else, each
    with a workspace: (function of keyword arguments, its result by itself)."""
    r = np.random.default_rng(n)
    lens = [[2000, 700], [1500, 1999], [64, 1800], [900, 1]][:n]
    kc, vc, sc, t = cache(r, [2000, 2000], 2, 16, 128, "int8", poison=False)
    pool = on_device(kc, vc, sc, t, "int8")
    calls = []
    for k in range(n):
        q, L = queries(r, 2, 8, 128, "bf16").to(DEV), dev(np.array(lens[k], np.int32))
        # (more parts than one: a workspace)
        calls.append(lambda q=q, L=L, k=k, **kw: tq4.kv8_paged_decode(
            q, *pool, L, num_splits=5 + k, **kw))
        q2, cu = queries(r, 8 + k, 8, 128, "bf16").to(DEV), dev(np.array([0, 4, 8 + k], np.int32))
        L2 = dev(np.maximum(lens[k], 16).astype(np.int32))
        calls.append(lambda q=q2, L=L2, cu=cu, k=k, **kw: tq4.kv8_paged_prefill(
            q, *pool, L, cu, 4 + k, **kw))
    wants = []
    for call in calls:
        torch.cuda.synchronize()
        wants.append(call())
        torch.cuda.synchronize()
    assert tq4.kv8_prefill_workspace_bytes(8, 2, 8, 2, 128, 16, t.shape[1], 4) > 0
    return list(zip(calls, wants))


def test_different_calls_at_once(tq4):
    """On streams of their own, by argument and by context, none waiting for another."""
    both = different_calls(tq4, 4)
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    outs = []
    for i in range(12):
        for k, (call, want) in enumerate(both):
            s = streams[(i + k) % 4]
            if i % 2:
                outs.append((call(stream=s), want))
            else:
                with torch.cuda.stream(s):
                    outs.append((call(), want))
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for out, want in outs)


def test_different_graphs_at_once(tq4):
    """Captured calls with workspaces of their own, replayed on two streams at a time
    between eager ones."""
    both = different_calls(tq4, 2)
    ws = [torch.full((1 << 24,), 255, dtype=torch.uint8, device=DEV) for _ in both]
    outs = [torch.empty_like(want) for _, want in both]
    graphs = []
    torch.cuda.synchronize()
    for (call, _), w, out in zip(both, ws, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(workspace=w, out=out)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for i in range(5):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        eager = []
        for k in range(len(graphs)):
            with torch.cuda.stream(streams[k]):
                graphs[k].replay()
            eager.append(both[k][0]())
        torch.cuda.synchronize()
        for (_, want), out, e in zip(both, outs, eager):
            assert torch.equal(out, want) and torch.equal(e, want)
