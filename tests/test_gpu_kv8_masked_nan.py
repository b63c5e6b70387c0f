"""NaN codes in the cache (the writer makes none; another writer may): a row that does
not see their token is as if they were not there, a row that sees it has a NaN in the
code's channel (values) or is NaN (keys)."""
import math

import numpy as np
import pytest
import torch

import kv8_reference as ref
from test_gpu_kv8_attention import DEV, cache, dev, on_device, queries

pytestmark = pytest.mark.gpu


def check(tq4, q, c, plain, lens, rows, tables_wide, **kw):
    """c: the cache with NaN codes; plain: the same with 448 in their places, from
    which the bound is taken (no code is larger)."""
    d = q.shape[2]
    cu = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    args = (lens, cu, "fp8", True, 1 / math.sqrt(d))
    want, _, _ = ref.attention(q.double().numpy(), *c, *args)
    _, off, _ = ref.attention(q.double().numpy(), *plain, *args)
    nan = np.isnan(want)
    assert nan.any() and not nan.all()
    kc, vc, sc, t = on_device(*c, "fp8")
    far = torch.full((len(lens), tables_wide), -1, dtype=torch.int32, device=DEV)
    far[:, :t.shape[1]] = t
    for table in (t, far):
        print("masked nan", tuple(q.shape), tuple(table.shape), list(rows), flush=True)
        out = tq4.kv8_paged_prefill(q.to(DEV), kc, vc, sc, table, dev(np.array(lens, np.int32)),
                                    dev(cu), max(rows), **kw)
        torch.cuda.synchronize()
        got = out.cpu()
        assert np.array_equal(got.isnan().numpy(), nan)
        ref.check(torch.nan_to_num(got, nan=0.0), np.where(nan, 0.0, want), off, q.dtype)


ROWS = [([17], [9]), ([70, 300], [70, 40]), ([130, 64, 33], [4, 3, 4]), ([700, 150], [200, 150])]


@pytest.mark.parametrize("plane", ["values", "keys"])
@pytest.mark.parametrize("d,H,G,S", [(64, 2, 1, 16), (128, 2, 4, 16), (256, 1, 8, 32),
                                     (128, 1, 5, 48), (64, 1, 16, 128), (256, 2, 3, 64)])
def test_nan_codes_at_the_causal_edge(tq4, d, H, G, S, plane):
    r = np.random.default_rng(d + H + G + S)
    for lens, rows in ROWS:
        kc, vc, sc, tables = cache(r, lens, H, S, d, "fp8", poison=False)
        plain = [kc, vc, sc, tables]
        nan = [kc.copy(), vc.copy(), sc, tables]
        for b, (n, k) in enumerate(zip(lens, rows)):
            # some tokens of the chunk, not its first: rows before each must not notice
            for t in sorted(set(r.integers(n - k + 1, n, 1 + k // 8))) if k > 1 else []:
                page, o = tables[b][t // S], t % S
                for h in range(H):
                    ch = r.integers(0, d, 2)
                    code = np.array([0x7F, 0xFF], np.uint8)
                    if plane == "values":
                        nan[1][page, h, o // 16, ch, o % 16] = code
                        plain[1][page, h, o // 16, ch, o % 16] = 0x7E
                    else:
                        nan[0][page, h, o, ch] = code
                        plain[0][page, h, o, ch] = 0x7E
        q = queries(r, sum(rows), H * G, d, "bf16", 0.5)
        check(tq4, q, nan, plain, lens, rows, 900000 // S)


def test_nan_values_in_parts(tq4):
    """The edge lies in the last of a tile's parts, or in a unit of its own."""
    r = np.random.default_rng(1)
    for d, G, lens, rows in ((128, 4, [2600], [70]), (64, 2, [2048 + 64], [64]),
                             (256, 2, [1500], [90]), (128, 4, [3000], [4])):
        kc, vc, sc, tables = cache(r, lens, 1, 16, d, "fp8", poison=False)
        plain, nan = [kc, vc, sc, tables], [kc, vc.copy(), sc, tables]
        t = lens[0] - rows[0] // 2
        nan[1][tables[0][t // 16], 0, 0, ::7, t % 16] = 0x7F
        plain[1] = vc.copy()
        plain[1][tables[0][t // 16], 0, 0, ::7, t % 16] = 0x7E
        check(tq4, queries(r, rows[0], G, d, "bf16", 0.5), nan, plain, lens, rows, 900000 // 16)
