"""Calls of the 8-bit cache's operators that their documentation allows, on the GPU."""
import numpy as np
import pytest
import torch

import kv8_reference as ref
from test_gpu_kv8_attention import cache, dev, on_device, queries

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_any_longer_max_query_len_means_the_rows(tq4):
    kc, vc, sc = tq4.kv8_cache(6, 2, 16, 64)
    k = torch.randn(70, 2, 64, device="cuda").bfloat16()
    tq4.kv8_reshape_and_cache(k, k, kc, vc, sc, torch.arange(70, dtype=torch.int32, device="cuda"))
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    q = torch.randn(70, 4, 64, device="cuda").bfloat16()
    args = (q, kc, vc, sc, i(0, 1, 2, 3, 4)[None], i(70), i(0, 70))
    want = tq4.kv8_paged_prefill(*args, 70)
    for longest in (71, 2 ** 31, 2 ** 32 + 4, 2 ** 70):
        assert torch.equal(tq4.kv8_paged_prefill(*args, longest), want)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_scale_that_is_no_number(tq4, d):
    """Every row that sees a token is NaN, whichever kernel takes the call."""
    r = np.random.default_rng(d)
    lens, rows = [50, 90], [20, 40]
    kc, vc, sc, tables = on_device(*cache(r, lens, 1, 16, d, "int8"), "int8")
    far = torch.full((2, 60000), -1, dtype=torch.int32, device=DEV)
    far[:, :tables.shape[1]] = tables
    L = dev(np.array(lens, np.int32))
    q = queries(r, 60, 2, d, "bf16").to(DEV)
    for t in (tables, far):
        assert tq4.kv8_paged_decode(q[:2], kc, vc, sc, t, L, scale=float("nan")).isnan().all()
        for n in (rows, [3, 2]):
            cu = dev(np.array([0, n[0], sum(n)], np.int32))
            out = tq4.kv8_paged_prefill(q[:sum(n)], kc, vc, sc, t, L, cu, max(n),
                                        scale=float("nan"))
            assert out.isnan().all()


def test_released_entries_that_name_no_page(tq4):
    """They go to the ring as they are (a released context's have to name pages): the
    rows of the request that gets one have slot -1, nothing else is touched, and the
    other pages are neither lost nor held twice."""
    B, S, M, P = 3, 16, 4, 8
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    ctx, ring, state = i(40, 0, 0), i(0, 1, 2, 3, 4, 5, 6, 7), i(0, 5)
    tables = torch.full((B, M), -1, dtype=torch.int32, device=DEV)
    tables[0, :3] = i(5, P + 9, 7)  # the middle page was taken away
    slots, cu, granted = torch.empty(64, dtype=torch.int32, device=DEV), i(0, 0, 0, 0), i(0, 0, 0)

    def step(new, release):
        c = dict(ctx=ctx, tables=tables, ring=ring, state=state)
        c = {k: v.cpu().numpy() for k, v in c.items()}
        tq4.paged_plan(ctx, i(*new), tables, ring, state, slots, cu, granted, S,
                       release=i(*release))
        want = ref.plan(c["ctx"], np.array(new), np.array(release), c["tables"], c["ring"],
                        c["state"], S, 64)
        got = dict(slots=slots, cu=cu, granted=granted, lens=ctx, state=state, tables=tables,
                   ring=ring)
        for k, g in got.items():
            assert np.array_equal(g.cpu().numpy(), want[k]), k
        return slots.cpu().numpy()

    step((0, 0, 0), (1, 0, 0))
    assert state.tolist() == [0, 8] and ring[5:].tolist() == [5, P + 9, 7]
    step((0, 60, 0), (0, 0, 0))
    got = step((0, 0, 60), (0, 0, 0))
    assert granted.tolist() == [0, 0, 60] and tables[2].tolist() == [4, 5, P + 9, 7]
    assert (got[:60] == -1).tolist() == [32 <= t < 48 for t in range(60)]
    kc, vc, sc = tq4.kv8_cache(P, 1, S, 64)
    k = torch.ones(64, 1, 64, dtype=torch.bfloat16, device=DEV)
    tq4.kv8_reshape_and_cache(k, k, kc, vc, sc, slots)
    assert (sc[0, :, 0] > 0).tolist() == [page in (4, 5, 7) for page in range(P)]
    out = tq4.kv8_paged_prefill(k[:60], kc, vc, sc, tables, ctx, cu, 60)
    assert torch.allclose(out.float(), torch.ones_like(out.float()), atol=2 ** -7)
