"""tq4_kv8_reshape_and_cache against the definition: every byte of the pools and
every scale, those that the call does not own included."""
import numpy as np
import pytest
import torch

import kv8_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def pools(r, P, H, S, d, code):
    kc = r.integers(0, 256, (P, H, S, d)).astype(np.uint8)
    vc = r.integers(0, 256, (P, H, S // 16, d, 16)).astype(np.uint8)
    sc = (2.0 ** r.integers(-9, 3, (2, P, H))).astype(np.float32)
    return kc, vc, sc


def activations(r, T, H, d, dtype, size=1.0):
    x = r.standard_normal((T, H, d)) * size * np.exp(r.standard_normal((T, 1, 1)))
    return torch.from_numpy(x).to(ref.TYPES[dtype])


def run(tq4, key, value, kc, vc, sc, slots, code, pad=0):
    """The call on copies; rows `pad` heads apart. Returns bytes and scales."""
    def rows(x):
        x = x.to(DEV)
        if not pad:
            return x
        wide = torch.full((x.shape[0], x.shape[1] + pad, x.shape[2]), float("nan"), dtype=x.dtype,
                          device=DEV)
        wide[:, pad // 2:pad // 2 + x.shape[1]] = x
        return wide[:, pad // 2:pad // 2 + x.shape[1]]
    g = lambda a: torch.from_numpy(a.copy()).to(DEV)  # noqa: E731
    dk, dv, ds = g(kc).view(ref.CODES[code]), g(vc).view(ref.CODES[code]), g(sc)
    print("write", tuple(key.shape), kc.shape, key.dtype, code, flush=True)
    tq4.kv8_reshape_and_cache(rows(key), rows(value), dk, dv, ds,
                              g(np.asarray(slots, np.int32)))
    torch.cuda.synchronize()
    return (dk.view(torch.uint8).cpu().numpy(), dv.view(torch.uint8).cpu().numpy(),
            ds.cpu().numpy())


def same(got, key, value, kc, vc, sc, slots, code):
    want = ref.write(key.float().numpy(), value.float().numpy(), kc, vc, sc, slots, code)
    for name, g, w in zip(("scales", "keys", "values"), (got[2], got[0], got[1]),
                          (want[2], want[0], want[1])):
        if name == "scales":
            g, w = g.view(np.uint32), w.astype(np.float32).view(np.uint32)
        assert np.array_equal(g, w), (name, (g != w).sum(), np.argwhere(g != w)[:4].tolist())


def prompt(r, P, S, starts):
    """Rows at consecutive places of distinct pages: [(start, rows), ..]."""
    free = list(r.permutation(P))
    slots = []
    for start, rows in starts:
        pages = [free.pop() for _ in range(-(-(start + rows) // S))]
        slots += [int(pages[i // S]) * S + i % S for i in range(start, start + rows)]
    return np.array(slots)


SHAPES = [(64, 1, 16), (64, 3, 32), (128, 8, 16), (128, 2, 48), (256, 2, 128), (128, 5, 64)]


@pytest.mark.parametrize("code", ["fp8", "int8"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d,H,S", SHAPES)
def test_writer(tq4, d, H, S, dtype, code):
    r = np.random.default_rng(d + 7 * H + S)
    starts = [(0, 1), (0, S), (3, 1), (S - 1, 2), (5, 2 * S), (0, 3 * S + 7), (S - 1, 1), (16, 16)
              if S > 16 else (1, 15)]
    slots = prompt(r, 40, S, starts)
    kc, vc, sc = pools(r, 40, H, S, d, code)
    k, v = activations(r, len(slots), H, d, dtype), activations(r, len(slots), H, d, dtype, 30)
    same(run(tq4, k, v, kc, vc, sc, slots, code), k, v, kc, vc, sc, slots, code)
    same(run(tq4, k, v, kc, vc, sc, slots, code, pad=2), k, v, kc, vc, sc, slots, code)


@pytest.mark.parametrize("code", ["fp8", "int8"])
def test_writer_decode_steps(tq4, code):
    """Rows of many sequences, one each, step after step into the same pages."""
    r = np.random.default_rng(5)
    B, H, S, d = 130, 2, 16, 128
    kc, vc, sc = pools(r, B + 3, H, S, d, code)
    pages = r.permutation(B + 3)[:B]
    at = r.integers(0, S, B)
    for step in range(4):
        slots = pages * S + (at + step) % S
        k, v = activations(r, B, H, d, "bf16", 4.0 ** step), activations(r, B, H, d, "bf16")
        got = run(tq4, k, v, kc, vc, sc, slots, code, pad=4)
        same(got, k, v, kc, vc, sc, slots, code)
        kc, vc, sc = got


@pytest.mark.parametrize("code", ["fp8", "int8"])
def test_writer_pads_order_and_repeats(tq4, code):
    """Slots outside the pool write nothing; offsets of a page in any order; of
    two rows for one slot the later one stays."""
    r = np.random.default_rng(6)
    H, S, d, P = 3, 32, 64, 12
    kc, vc, sc = pools(r, P, H, S, d, code)
    a = 4 * S + r.permutation(S)              # a whole page, shuffled
    b = 7 * S + np.array([9, 8, 30, 9, 9, 2])  # repeats
    c = 2 * S + np.concatenate([np.arange(S), [0, 5, 0]])  # more rows than a page has
    slots = np.concatenate([[-1, -5, P * S, 2 ** 31 - 1], a, [-1], b, c, [-1, 9 * S + 3]])
    k, v = activations(r, len(slots), H, d, "fp16"), activations(r, len(slots), H, d, "fp16")
    same(run(tq4, k, v, kc, vc, sc, slots, code), k, v, kc, vc, sc, slots, code)
    same(run(tq4, k[:4], v[:4], kc, vc, sc, slots[:4], code), k[:4], v[:4], kc, vc, sc, slots[:4],
         code)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("code", ["fp8", "int8"])
def test_writer_values_at_the_ends(tq4, code, dtype):
    """Zeros, infinities, NaN, the largest and the smallest magnitudes, those at
    the borders of a scale and ties of the rounding."""
    r = np.random.default_rng(7)
    H, S, d = 1, 16, 64
    info = torch.finfo(ref.TYPES[dtype])
    rows = []
    for x in (0.0, float("inf"), float("-inf"), float("nan"), info.max, info.tiny,
              info.tiny * info.eps, 448.0, 449.0, 450.0, 127.0, 127.5, 128.0, 254.0, 255.0, 1.0):
        row = torch.zeros(d)
        row[3] = x
        row[7] = -x / 2
        row[8:40] = torch.linspace(-2.5, 2.5, 32) * (1 if x != x or abs(x) > 1e30 else abs(x) / 3)
        rows.append(row)
    x = torch.stack(rows).to(ref.TYPES[dtype])[:, None]
    T = len(rows)
    kc, vc, sc = pools(r, T + 2, H, S, d, code)
    odd = np.array([0.0, np.nan, np.inf, -1.0, 0.3, 1e-38, 3.0, 1e30], np.float32)
    sc = odd[np.arange(sc.size) % 8].reshape(sc.shape)
    for off in (0, 5):
        slots = np.arange(T) * S + off
        same(run(tq4, x, x, kc, vc, sc, slots, code), x, x, kc, vc, sc, slots, code)
    slots = np.arange(T)  # all in one page
    same(run(tq4, x, x, kc, vc, sc, slots, code), x, x, kc, vc, sc, slots, code)


def test_writer_one_row_views(tq4):
    """One row, whose row stride means nothing, and a long run in large pages."""
    r = np.random.default_rng(8)
    kc, vc, sc = pools(r, 5, 2, 1024, 128, "fp8")
    k = activations(r, 1, 2, 128, "bf16")
    same(run(tq4, k, k, kc, vc, sc, [1024 + 77], "fp8"), k, k, kc, vc, sc, [1024 + 77], "fp8")
    slots = 3000 + np.arange(2000)
    k, v = activations(r, 2000, 2, 128, "bf16"), activations(r, 2000, 2, 128, "bf16")
    same(run(tq4, k, v, kc, vc, sc, slots, "fp8"), k, v, kc, vc, sc, slots, "fp8")


@pytest.mark.parametrize("T", [1025, 2500, 5000])
def test_writer_many_rows(tq4, T):
    """Sizes at which rows are dealt to waves in larger windows: prompt chunks
    between single rows, with pads."""
    r = np.random.default_rng(T)
    S, H, d = 16, 2, 64
    starts, left = [], T
    while left > 0:
        n = 1 if r.random() < 0.5 else int(r.integers(2, 90))
        starts.append((int(r.integers(0, S)), min(n, left)))
        left -= min(n, left)
    P = sum(-(-(a + n) // S) for a, n in starts) + 1
    slots = prompt(r, P, S, starts)
    slots[r.random(T) < 0.02] = -1
    # a pad inside a page's rows would part them: give such pages' later rows up
    seen, last = set(), None
    for i, s in enumerate(slots):
        page = s // S if s >= 0 else None
        if page is not None and page != last and page in seen:
            slots[i] = -1
            page = None
        if page is not None:
            seen.add(page)
        last = page
    kc, vc, sc = pools(r, P, H, S, d, "int8")
    k, v = activations(r, T, H, d, "bf16"), activations(r, T, H, d, "bf16")
    same(run(tq4, k, v, kc, vc, sc, slots, "int8", pad=6), k, v, kc, vc, sc, slots, "int8")
