"""Calls of the 8-bit cache's operators that their documentation allows, on the GPU."""
import pytest
import torch

pytestmark = pytest.mark.gpu


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
