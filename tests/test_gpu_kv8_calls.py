"""Calls of the 8-bit cache's operators that their documentation allows, on the GPU."""
import numpy as np
import pytest
import torch

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
