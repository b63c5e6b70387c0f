"""The attention over the 8-bit paged cache against the definition in 64 bits,
element by element within the bound that kv8_reference.attention derives."""
import math

import numpy as np
import pytest
import torch

import kv8_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def cache(r, lens, H, S, d, code, extra=2, width=None, spread=3, poison=True):
    """Pools whose pages hold random codes; bytes past the contexts, and pages of
    no sequence, hold every byte (NaN codes too) when `poison`."""
    held = [-(-n // S) for n in lens]
    P = sum(held) + extra
    M = max(max(held, default=0), 1) if width is None else width
    order = r.permutation(P)
    tables = np.full((len(lens), M), -1, np.int32)
    any_byte = r.integers(0, 256, (2, P, H, S, d)).astype(np.uint8)
    if code == "fp8":
        fine = ref.to_codes(r.standard_normal((2, P, H, S, d)) * 60, code)
    else:
        fine = (r.integers(-127, 128, (2, P, H, S, d))).astype(np.int8).view(np.uint8)
    x = any_byte if poison else fine.copy()
    at = 0
    for b, n in enumerate(lens):
        for i in range(held[b]):
            page = order[at]
            tables[b, i] = page
            live = min(S, n - i * S)
            x[:, page, :, :live] = fine[:, page, :, :live]
            at += 1
    sc = (2.0 ** r.integers(-9, -9 + spread, (2, P, H))).astype(np.float32)
    v = np.ascontiguousarray(x[1].reshape(P, H, S // 16, 16, d).transpose(0, 1, 2, 4, 3))
    return np.ascontiguousarray(x[0]), v, sc, tables


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def queries(r, rows, Hq, d, dtype, size=1.0):
    return torch.from_numpy(r.standard_normal((rows, Hq, d)) * size).to(ref.TYPES[dtype])


def wide(x, pad):
    """x as a slice of rows `pad` heads longer, the rest NaN."""
    w = torch.full((x.shape[0], x.shape[1] + pad, x.shape[2]), float("nan"), dtype=x.dtype,
                   device=DEV)
    w[:, :x.shape[1]] = x
    return w[:, :x.shape[1]]


def on_device(kc, vc, sc, tables, code):
    return (dev(kc).view(ref.CODES[code]), dev(vc).view(ref.CODES[code]), dev(sc), dev(tables))


def decode(tq4, q, c, lens, code, pad=0, **kw):
    kc, vc, sc, tables = on_device(*c, code)
    qd = q.to(DEV)
    print("decode", tuple(q.shape), kc.shape, q.dtype, code, list(lens)[:8], kw, flush=True)
    out = tq4.kv8_paged_decode(wide(qd, pad) if pad else qd, kc, vc, sc, tables,
                               dev(np.asarray(lens, np.int32)), **kw)
    torch.cuda.synchronize()
    return out


def check_decode(tq4, q, c, lens, code, scale=None, pad=0, **kw):
    kc, vc, sc, tables = c
    d = q.shape[2]
    want, off, _ = ref.attention(q.double().numpy(), kc, vc, sc, tables, lens,
                                 np.arange(len(lens) + 1), code, False,
                                 1 / math.sqrt(d) if scale is None else scale)
    if scale is not None:
        kw["scale"] = scale
    out = decode(tq4, q, c, lens, code, pad, **kw)
    print("of the bound:", ref.check(out, want, off, q.dtype))
    S = kc.shape[2]
    if "num_splits" not in kw and max(lens) <= tables.shape[1] * S:
        # in a table of many pages the sequences are cut, or streamed
        far = np.full((len(lens), 60000 // S), -1, np.int32)
        far[:, :tables.shape[1]] = tables
        ref.check(decode(tq4, q, (kc, vc, sc, far), lens, code, pad, **kw), want, off, q.dtype)
    return out


LENS = [[1], [0], [15, 16, 17], [63, 64, 65, 0, 1], [255, 256, 257], [513, 1, 1040], [2049]]


@pytest.mark.parametrize("code", ["fp8", "int8"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d,H,G,S", [(64, 2, 1, 16), (128, 2, 4, 16), (256, 1, 16, 32),
                                     (128, 1, 5, 48), (64, 3, 8, 128), (256, 2, 3, 64)])
def test_decode(tq4, d, H, G, S, dtype, code):
    r = np.random.default_rng(d + H + G + S)
    for lens in LENS:
        c = cache(r, lens, H, S, d, code)
        check_decode(tq4, queries(r, len(lens), H * G, d, dtype, 3.0), c, lens, code,
                     pad=2 if S == 16 else 0)


@pytest.mark.parametrize("K", [1, 2, 3, 7, 64, 256])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_decode_splits(tq4, d, K):
    """Any count of splits, more than there are tokens among them."""
    r = np.random.default_rng(K + d)
    lens = [1500, 0, 1, 200, 64 * 7, 999]
    c = cache(r, lens, 2, 16, d, "fp8")
    q = queries(r, len(lens), 8, d, "bf16", 2.0)
    n = tq4.kv8_decode_workspace_bytes(len(lens), 8, 2, d, 16, c[3].shape[1], K)
    ws = torch.full((n,), 255, dtype=torch.uint8, device=DEV) if n else None
    out = check_decode(tq4, q, c, lens, "fp8", num_splits=K, workspace=ws)
    given = torch.full_like(out, float("nan"))
    again = decode(tq4, q, c, lens, "fp8", num_splits=K, out=given)
    assert again is given and torch.equal(given, out)


def test_decode_pages_that_name_nothing(tq4):
    """Entries outside the pool contribute nothing; a sequence of them alone is 0;
    a context past the table is cut at it."""
    r = np.random.default_rng(1)
    for S, code in ((16, "fp8"), (64, "int8")):
        lens = [5 * S, 3 * S + 1, 6 * S - 3, S, 9 * S]
        c = cache(r, lens[:4] + [6 * S], 2, S, 128, code)
        t = c[3]
        t[0, 1], t[0, 4] = -1, 10 ** 6
        t[1, 3] = c[0].shape[0]
        t[2, 0] = -2 ** 31
        t[3, 0] = -1
        out = check_decode(tq4, queries(r, 5, 8, 128, "bf16"), c, lens, code)
        assert (out[3] == 0).all()
    c = cache(r, [100, 50], 1, 16, 64, "fp8")
    out = check_decode(tq4, queries(r, 2, 1, 64, "bf16"), c, [-4, 50], "fp8")
    assert (out[0] == 0).all()


@pytest.mark.parametrize("code", ["fp8", "int8"])
def test_decode_scales_far_apart(tq4, code):
    """Scales of keys and values that differ by many powers of two, no powers of
    two, out of range; scores that grow along the context."""
    r = np.random.default_rng(2)
    lens = [1000, 333]
    c = list(cache(r, lens, 2, 16, 128, code))
    sc = c[2]
    sc[1] = (2.0 ** r.integers(-40, 40, sc[1].shape)).astype(np.float32)
    check_decode(tq4, queries(r, 2, 8, 128, "bf16"), c, lens, code)
    sc[:] = (r.random(sc.shape) + 0.01).astype(np.float32) * 0.05
    check_decode(tq4, queries(r, 2, 8, 128, "fp16"), c, lens, code)
    # later pages win by far, so the running maximum moves every time
    for b in range(2):
        for i, p in enumerate(c[3][b][c[3][b] >= 0]):
            sc[0, p] = 2.0 ** -9 * 1.3 ** i
            sc[1, p] = 2.0 ** (-9 - i % 7)
    check_decode(tq4, queries(r, 2, 8, 128, "bf16"), c, lens, code)
    sc[0], sc[1] = 2.0 ** -9, 0.0  # read as 2^-100
    out = decode(tq4, queries(r, 2, 8, 128, "bf16"), c, lens, code)
    assert (out.float().abs() < 1e-25).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_decode_queries_of_every_size(tq4, dtype):
    """Rows of tiny and huge magnitude, of zeros; one with a NaN or an infinity
    is its own affair. A scale that is negative, zero or large."""
    r = np.random.default_rng(3)
    lens = [300, 40]
    c = cache(r, lens, 1, 16, 64, "fp8", spread=1)
    q = queries(r, 2, 8, 64, dtype).double()
    q[:, 1] = 0
    q[:, 2] *= 2.0 ** -12 if dtype == "fp16" else 2.0 ** -120
    q[:, 3] *= 2.0 ** 9 if dtype == "fp16" else 2.0 ** 40
    q[:, 4, 5] = 2.0 ** 12
    q[:, 5, ::2] *= 2.0 ** -9
    q = q.to(ref.TYPES[dtype])
    if dtype == "bf16":
        q[:, 3] *= 2.0 ** -38
    for scale in (None, -0.2, 0.0, 1.0):
        check_decode(tq4, q, c, lens, "fp8", scale=scale)
    bad = q.clone()
    bad[0, 0, 3], bad[1, 6, 1] = float("nan"), float("inf")
    out, fine = decode(tq4, bad, c, lens, "fp8"), decode(tq4, q, c, lens, "fp8")
    keep = torch.ones(2, 8, dtype=torch.bool)
    keep[0, 0] = keep[1, 6] = False
    assert torch.equal(out[keep], fine[keep]) and out[0, 0].isnan().all()


def test_decode_offsets_past_32_bits(tq4):
    """A pool of more than 4 GiB a plane, its sequences at the far end."""
    H, S, d = 8, 128, 256
    P = (2 ** 32) // (H * S * d) + 40
    r = np.random.default_rng(4)
    kc = torch.full((P, H, S, d), 0x7F, dtype=torch.uint8, device=DEV)
    vc = torch.full((P, H, S // 16, d, 16), 0x7F, dtype=torch.uint8, device=DEV)
    sc = torch.full((2, P, H), 2.0 ** -8, device=DEV)
    lens = [300, 129]
    small = cache(r, lens, H, S, d, "fp8", extra=0, poison=False)
    n = small[0].shape[0]
    kc[P - n:], vc[P - n:] = dev(small[0]), dev(small[1])
    sc[:, P - n:] = dev(small[2])
    q = queries(r, 2, 16, d, "bf16")
    want, off, _ = ref.attention(q.double().numpy(), *small, lens, [0, 1, 2], "fp8", False, 1 / 16)
    t = np.where(small[3] >= 0, small[3] + P - n, -1).astype(np.int32)
    out = tq4.kv8_paged_decode(q.to(DEV), kc.view(ref.CODES["fp8"]), vc.view(ref.CODES["fp8"]), sc,
                               dev(t), dev(np.array(lens, np.int32)))
    ref.check(out, want, off, q.dtype)
    # the writer, there too
    k = queries(r, 3, H, d, "bf16")
    slots = np.array([(P - 1) * S, (P - 1) * S + 1, (P - 2) * S + 5], np.int32)
    tail = [x[P - 2:].cpu().numpy() for x in (kc, vc)] + [sc[:, P - 2:].cpu().numpy()]
    tq4.kv8_reshape_and_cache(k.to(DEV), k.to(DEV), kc.view(ref.CODES["fp8"]),
                              vc.view(ref.CODES["fp8"]), sc, dev(slots))
    w = ref.write(k.float().numpy(), k.float().numpy(), *tail, slots - (P - 2) * S, "fp8")
    assert np.array_equal(kc[P - 2:].cpu().numpy(), w[0])
    assert np.array_equal(vc[P - 2:].cpu().numpy(), w[1])
    assert np.array_equal(sc[:, P - 2:].cpu().numpy(), w[2])


# ------------------------------------------------------------ several rows
def check_prefill(tq4, q, c, lens, rows, code, causal, pad=0, max_q=None, scale=None, **kw):
    """Rows behind the last sequence have to stay as they were."""
    kc, vc, sc, tables = c
    d = q.shape[2]
    cu = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    want, off, done = ref.attention(q.double().numpy(), kc, vc, sc, tables, lens, cu, code, causal,
                                    1 / math.sqrt(d) if scale is None else scale, max_q)
    kw["scale"] = scale
    dk, dv, ds, dt = on_device(kc, vc, sc, tables, code)
    qd = q.to(DEV)
    at = torch.from_numpy(done)
    # a table of many pages more takes more than a few rows to the kernel for prompts
    S = kc.shape[2]
    far = torch.full((len(lens), max(900000 // S, dt.shape[1])), -1, dtype=torch.int32, device=DEV)
    far[:, :dt.shape[1]] = dt
    for t in (dt, far) if max(lens) <= dt.shape[1] * S else (dt,):
        out = torch.full(q.shape, 77.0, dtype=q.dtype, device=DEV)
        print("prefill", tuple(q.shape), kc.shape, tuple(t.shape), q.dtype, code, causal,
              list(lens)[:6], list(rows)[:6], flush=True)
        got = tq4.kv8_paged_prefill(wide(qd, pad) if pad else qd, dk, dv, ds, t,
                                    dev(np.asarray(lens, np.int32)), dev(cu),
                                    max(rows, default=0) if max_q is None else max_q,
                                    causal=causal, out=out, **kw)
        torch.cuda.synchronize()
        assert got is out
        assert (out[torch.from_numpy(~done).to(DEV)] == 77.0).all()
        print("of the bound:", ref.check(out[at.to(DEV)], want[done], off[done], q.dtype))
    return out


ROWS = [([1], [1]), ([5, 5], [5, 5]), ([17, 130, 64], [1, 7, 64]), ([300, 33], [100, 33]),
        ([0, 40, 700], [3, 0, 5]), ([20, 257], [33, 257]), ([129, 64, 1, 900], [65, 3, 1, 200])]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("code,dtype", [("fp8", "bf16"), ("int8", "fp16"), ("fp8", "fp16"),
                                        ("int8", "bf16")])
@pytest.mark.parametrize("d,H,G,S", [(64, 2, 1, 16), (128, 2, 4, 16), (256, 1, 16, 32),
                                     (128, 1, 5, 48), (64, 1, 8, 128), (256, 2, 3, 64)])
def test_prefill(tq4, d, H, G, S, code, dtype, causal):
    r = np.random.default_rng(d + H + G + S)
    for k, (lens, rows) in enumerate(ROWS):
        c = cache(r, lens, H, S, d, code)
        tail = k % 3
        q = queries(r, sum(rows) + tail, H * G, d, dtype, 2.0)
        check_prefill(tq4, q, c, lens, rows, code, causal, pad=3 * (k % 2))


@pytest.mark.parametrize("causal", [True, False])
def test_prefill_few_rows_of_long_contexts(tq4, causal):
    """Drafted tokens: the contexts are split and joined."""
    r = np.random.default_rng(11)
    for d, G, rows, lens in ((128, 4, [4] * 5, [3000, 1, 700, 5000, 64]),
                             (256, 8, [2, 1, 0, 2], [4000, 900, 5, 1300]),
                             (64, 2, [8, 3, 7], [2500, 2600, 70])):
        lens = [max(a, b) for a, b in zip(lens, rows)]
        c = cache(r, lens, 2, 16, d, "fp8")
        check_prefill(tq4, queries(r, sum(rows), 2 * G, d, "bf16"), c, lens, rows, "fp8", causal)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d,G,rows,lens", [(128, 4, [70, 20], [2600, 1]), (64, 2, [100], [4100]),
                                           (256, 8, [40, 9, 0], [1500, 700, 300]),
                                           (128, 1, [300, 129, 1], [1800, 2000, 1100])])
def test_prefill_parts(tq4, d, G, rows, lens, causal):
    """Row tiles too few for the GPU: their contexts are cut into parts and joined."""
    r = np.random.default_rng(d + G)
    lens = [max(a, b) for a, b in zip(lens, rows)]
    c = cache(r, lens, 1, 32, d, "int8")
    assert tq4.kv8_prefill_workspace_bytes(sum(rows), len(rows), G, 1, d, 32, 900000 // 32,
                                           max(rows)) > 0
    check_prefill(tq4, queries(r, sum(rows) + 1, G, d, "fp16"), c, lens, rows, "int8", causal)


@pytest.mark.parametrize("d,causal", [(64, True), (128, False), (256, True)])
def test_prefill_of_many_rows(tq4, d, causal):
    """Row tiles enough for the GPU: nothing is cut."""
    r = np.random.default_rng(d)
    lens, rows = [1000, 555, 33, 700], [900, 555, 1, 77]
    H = 32 if d < 256 else 24
    c = cache(r, lens, H, 16, d, "fp8")
    assert tq4.kv8_prefill_workspace_bytes(sum(rows), 4, H, H, d, 16, c[3].shape[1],
                                           max(rows)) == 0
    check_prefill(tq4, queries(r, sum(rows) + 1, H, d, "bf16"), c, lens, rows, "fp8", causal)


def test_prefill_wrong_lengths_stay_inside(tq4):
    """max_query_len below a sequence's rows: the rows past it are left; pages
    that name nothing in the middle; contexts past the table."""
    r = np.random.default_rng(12)
    lens, rows = [200, 90, 300], [50, 20, 33]
    c = cache(r, lens, 2, 16, 128, "fp8")
    c[3][0, 2] = c[3][2, 18] = -1
    c[3][1, 0] = 10 ** 7
    q = queries(r, sum(rows) + 4, 8, 128, "bf16")
    check_prefill(tq4, q, c, lens, rows, "fp8", True)
    check_prefill(tq4, q, c, lens, rows, "fp8", False, max_q=17)
    check_prefill(tq4, q, c, [200, 90, 10 ** 6], rows, "fp8", True, max_q=3)


def test_prefill_row_ranges(tq4):
    """Rows before the first sequence and past num_rows, ranges without rows."""
    r = np.random.default_rng(15)
    lens, cu = [300, 50, 120, 90], np.array([7, 60, 60, 180, 200], np.int32)
    for d, H in ((64, 1), (128, 2), (256, 1)):
        c = cache(r, lens, H, 16, d, "int8")
        kc, vc, sc, t = on_device(*c, "int8")
        far = torch.full((4, 60000), -1, dtype=torch.int32, device=DEV)
        far[:, :t.shape[1]] = t
        q = queries(r, 200, 4 * H, d, "bf16")
        want, off, done = ref.attention(q.double().numpy(), *c, lens, cu, "int8", True,
                                        1 / math.sqrt(d))
        for rows in (200, 150, 60, 8, 7):
            for table in (t, far):
                print("ranges", d, rows, tuple(table.shape), flush=True)
                out = torch.full((rows, 4 * H, d), 77.0, dtype=q.dtype, device=DEV)
                tq4.kv8_paged_prefill(q[:rows].to(DEV), kc, vc, sc, table,
                                      dev(np.array(lens, np.int32)), dev(cu), 120, out=out)
                torch.cuda.synchronize()
                assert (out[torch.from_numpy(~done[:rows]).to(DEV)] == 77.0).all()
                at = torch.from_numpy(done[:rows]).to(DEV)
                ref.check(out[at], want[:rows][done[:rows]], off[:rows][done[:rows]], q.dtype)


@pytest.mark.parametrize("S,d", [(1024, 64), (1024, 256), (80, 128), (16, 256), (512, 128)])
def test_page_sizes(tq4, S, d):
    """Pages of many strips and of odd counts of them, written and attended over."""
    r = np.random.default_rng(S + d)
    lens = [S + 17, 5, 2 * S]
    kc, vc, sc = tq4.kv8_cache(9, 2, S, d)
    order = r.permutation(9)
    tables = np.full((3, 3), -1, np.int32)
    slots, at = [], 0
    for b, n in enumerate(lens):
        for i in range(-(-n // S)):
            tables[b, i] = order[at]
            at += 1
        slots += [tables[b, i // S] * S + i % S for i in range(n)]
    k, v = queries(r, sum(lens), 2, d, "bf16"), queries(r, sum(lens), 2, d, "bf16", 5.0)
    tq4.kv8_reshape_and_cache(k.to(DEV), v.to(DEV), kc, vc, sc, dev(np.array(slots, np.int32)))
    raw = [x.view(torch.uint8).cpu().numpy() for x in (kc, vc)] + [sc.cpu().numpy()]
    empty = [np.zeros_like(x) for x in raw]
    want = ref.write(k.float().numpy(), v.float().numpy(), *empty, np.array(slots), "fp8")
    assert all(np.array_equal(a, b) for a, b in zip(raw, want))
    check_decode(tq4, queries(r, 3, 8, d, "bf16"), (*raw, tables), lens, "fp8")
    check_prefill(tq4, queries(r, 70, 4, d, "bf16"), (*raw, tables), lens, [60, 1, 9], "fp8", True)


def test_nothing_to_do(tq4):
    """No sequences, no rows, no tokens: nothing is launched, nothing refused."""
    kc, vc, sc = tq4.kv8_cache(3, 2, 16, 64)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=DEV)  # noqa: E731
    rows = lambda n, h: torch.ones((n, h, 64), dtype=torch.bfloat16, device=DEV)  # noqa: E731
    tq4.kv8_reshape_and_cache(rows(0, 2), rows(0, 2), kc, vc, sc, i32(0))
    assert tq4.kv8_paged_decode(rows(0, 4), kc, vc, sc, i32(0, 2), i32(0)).shape == (0, 4, 64)
    none = tq4.kv8_paged_prefill(rows(0, 4), kc, vc, sc, i32(2, 2), i32(2), i32(3), 5)
    assert none.shape == (0, 4, 64)
    out = rows(3, 4)
    tq4.kv8_paged_prefill(rows(3, 4), kc, vc, sc, i32(2, 2), i32(2), i32(3), 0, out=out)
    tq4.kv8_paged_prefill(rows(3, 4), kc, vc, sc, i32(0, 2), i32(0), i32(1), 3, out=out)
    assert (out == 1).all() and (sc == 0).all()


@pytest.mark.parametrize("code", ["fp8", "int8"])
def test_prefill_scales_far_apart(tq4, code):
    r = np.random.default_rng(13)
    lens, rows = [700, 333], [150, 333]
    c = cache(r, lens, 1, 16, 128, code)
    sc = c[2]
    sc[1] = (2.0 ** r.integers(-40, 40, sc[1].shape)).astype(np.float32)
    check_prefill(tq4, queries(r, 483, 4, 128, "bf16"), c, lens, rows, code, True)
    for b in range(2):
        for i, p in enumerate(c[3][b][c[3][b] >= 0]):
            sc[0, p] = 2.0 ** -9 * 1.2 ** i
            sc[1, p] = 2.0 ** (-9 - i % 7)
    check_prefill(tq4, queries(r, 483, 4, 128, "fp16"), c, lens, rows, code, True)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_prefill_queries_of_every_size(tq4, dtype):
    """Scales that are negative, zero or large; rows of zeros, of tiny and huge
    magnitude; a row with a NaN or an infinity is its own affair."""
    r = np.random.default_rng(14)
    lens, rows = [300, 129], [120, 40]
    for d in (64, 128, 256):
        c = cache(r, lens, 1, 16, d, "fp8", spread=1)
        q = queries(r, 160, 4, d, dtype).double()
        q[7] = 0
        q[8] *= 2.0 ** -12 if dtype == "fp16" else 2.0 ** -120
        q[9] *= 2.0 ** 9 if dtype == "fp16" else 2.0 ** 20
        q = q.to(ref.TYPES[dtype])
        for scale in (-0.2, 0.0, 1.0):
            check_prefill(tq4, q, c, lens, rows, "fp8", True, scale=scale)
        kc, vc, sc, t = on_device(*c, "fp8")
        L, cu = dev(np.array(lens, np.int32)), dev(np.array([0, 120, 160], np.int32))
        far = torch.full((2, 50000), -1, dtype=torch.int32, device=DEV)
        far[:, :t.shape[1]] = t
        bad = q.clone()
        bad[3, 1, 5], bad[130, 2, 0] = float("nan"), float("inf")
        keep = torch.ones(160, 4, dtype=torch.bool)
        keep[3, 1] = keep[130, 2] = False
        for table in (t, far):
            print("bad rows", d, tuple(table.shape), flush=True)
            fine = tq4.kv8_paged_prefill(q.to(DEV), kc, vc, sc, table, L, cu, 120)
            out = tq4.kv8_paged_prefill(bad.to(DEV), kc, vc, sc, table, L, cu, 120)
            assert torch.equal(out.cpu()[keep], fine.cpu()[keep])
            assert out[3, 1].isnan().all()


# ------------------------------------------------------------- a step of all
@pytest.mark.parametrize("code,dtype", [("fp8", "bf16"), ("int8", "fp16")])
def test_steps_of_plan_write_attend(tq4, code, dtype):
    """Continuous batching from an empty pool: every step plans, writes and
    attends on the GPU; each step's outputs are held against attention over the
    step's own cache."""
    r = np.random.default_rng(20)
    B, H, G, S, d, M, P = 9, 2, 4, 16, 64, 10, 60
    kc, vc, sc = tq4.kv8_cache(P, H, S, d, ref.CODES[code])
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=DEV)  # noqa: E731
    ctx, tables = i32(B), i32(B, M) - 1
    ring, state = dev(r.permutation(P).astype(np.int32)), dev(np.array([0, P], np.int32))
    cu, granted = i32(B + 1), i32(B)
    kept = {}
    for step in range(8):
        new = r.integers(0, 60, B) if step in (0, 4) else np.ones(B, int)
        release = (r.random(B) < 0.25).astype(np.int32) if step > 2 else np.zeros(B, np.int32)
        T = int(new.sum()) + 3
        slots, pos = i32(T), i32(T)
        tq4.paged_plan(ctx, dev(new.astype(np.int32)), tables, ring, state, slots, cu, granted, S,
                       release=dev(release), positions=pos)
        qkv = torch.randn((T, (G + 2) * H, d), device=DEV).to(ref.TYPES[dtype])
        q, k, v = qkv[:, :G * H], qkv[:, G * H:(G + 1) * H], qkv[:, (G + 1) * H:]
        tq4.kv8_reshape_and_cache(k, v, kc, vc, sc, slots)
        out = tq4.kv8_paged_prefill(q, kc, vc, sc, tables, ctx, cu, int(new.max()))
        g = granted.cpu().numpy()
        assert step > 0 or (g == new).any()
        raw = [x.view(torch.uint8).cpu().numpy() for x in (kc, vc)] + [sc.cpu().numpy()]
        lens = ctx.cpu().numpy()
        want, off, _ = ref.attention(q.double().cpu().numpy(), *raw, tables.cpu().numpy(), lens,
                                     cu.cpu().numpy(), code, True, 1 / math.sqrt(d))
        ok = np.repeat(np.concatenate([g == new, [False]]), np.concatenate([new, [3]]))
        ref.check(out[torch.from_numpy(ok).to(DEV)], want[ok], off[ok], q.dtype)
        if (new == 1).all():
            one = tq4.kv8_paged_decode(q[:B], kc, vc, sc, tables, ctx)
            ref.check(one[torch.from_numpy(ok[:B]).to(DEV)], want[:B][ok[:B]], off[:B][ok[:B]],
                      q.dtype)
        # the cache holds the step's keys: within half a code's step of them
        s = slots.cpu().numpy()
        for t in np.nonzero(s >= 0)[0][:20]:
            page, o = s[t] // S, s[t] % S
            held = ref.code_values(raw[0][page, :, o], code) * raw[2][0, page][:, None]
            x = k[t].double().cpu().numpy()
            step_size = (np.maximum(np.abs(x) * 2.0 ** -4, raw[2][0, page][:, None] * 2.0 ** -10)
                         if code == "fp8" else raw[2][0, page][:, None] / 2)
            assert (np.abs(held - x) <= step_size).all()
        kept[step] = int((s >= 0).sum())
    assert sum(kept.values()) > 200


def test_torch_ops(tq4):
    """The registered operators give the entry points' results."""
    r = np.random.default_rng(30)
    ops, lens = torch.ops.tq4, [70, 1]
    kc, vc, sc = tq4.kv8_cache(12, 1, 16, 64)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=DEV)  # noqa: E731
    ctx, tables, ring = i32(2), i32(2, 6), dev(r.permutation(12).astype(np.int32))
    slots, pos, cu, granted = i32(73), i32(73), i32(3), i32(2)
    ops.paged_plan(ctx, dev(np.array(lens, np.int32)), None, tables, ring,
                   dev(np.array([0, 12], np.int32)), slots, pos, cu, granted, 16)
    assert ctx.tolist() == lens == granted.tolist() and cu.tolist() == [0, 70, 71]
    k, v = queries(r, 73, 1, 64, "fp16").to(DEV), queries(r, 73, 1, 64, "fp16").to(DEV)
    ops.kv8_reshape_and_cache(k, v, kc, vc, sc, slots)
    q = queries(r, 73, 2, 64, "fp16").to(DEV)
    out = ops.kv8_paged_prefill(q, kc, vc, sc, tables, ctx, cu, 70, True, 0.0)
    want = tq4.kv8_paged_prefill(q, kc, vc, sc, tables, ctx, cu, 70)
    assert torch.equal(out[:71], want[:71]) and (out[71:] == 0).all()
    assert torch.equal(ops.kv8_paged_decode(q[:2], kc, vc, sc, tables, ctx, 2, 0.3),
                       tq4.kv8_paged_decode(q[:2], kc, vc, sc, tables, ctx, num_splits=2, scale=0.3))


def test_captured_step(tq4):
    """A captured step (write, decode, split and not), replayed with eager work
    between, gives the eager bits every time; two graphs have their own workspaces."""
    r = np.random.default_rng(21)
    lens = [900, 33, 500]
    c = cache(r, lens, 2, 16, 128, "fp8", poison=False)
    kc, vc, sc, tables = on_device(*c, "fp8")
    L = dev(np.array(lens, np.int32))
    slots = dev(np.array([c[3][b][(n - 1) // 16] * 16 + (n - 1) % 16 for b, n in enumerate(lens)],
                         np.int32))
    q, k = queries(r, 3, 8, 128, "bf16").to(DEV), queries(r, 3, 2, 128, "bf16").to(DEV)
    graphs = []
    for K in (1, 4):
        n = tq4.kv8_decode_workspace_bytes(3, 8, 2, 128, 16, tables.shape[1], K)
        ws = torch.empty(max(n, 16), dtype=torch.uint8, device=DEV)
        out = torch.empty_like(q)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            tq4.kv8_reshape_and_cache(k, k, kc, vc, sc, slots)
            tq4.kv8_paged_decode(q, kc, vc, sc, tables, L, out=out, workspace=ws, num_splits=K)
        graphs.append((K, g, out, ws))
    for i in range(4):
        q.copy_(queries(r, 3, 8, 128, "bf16"))
        k.copy_(queries(r, 3, 2, 128, "bf16"))
        for K, g, out, _ in graphs:
            out.zero_()
            g.replay()
            eager = tq4.kv8_paged_decode(q, kc, vc, sc, tables, L, num_splits=K)
            torch.cuda.synchronize()
            assert torch.equal(out, eager)


def test_captured_prefill(tq4):
    """Captured prefills, in parts and streamed, replayed with eager work between."""
    r = np.random.default_rng(23)
    lens, rows = [2100, 1500], [100, 30]
    c = cache(r, lens, 1, 16, 128, "fp8", width=6000)
    kc, vc, sc, tables = on_device(*c, "fp8")
    L = dev(np.array(lens, np.int32))
    for n in (rows, [3, 4]):
        cu = dev(np.concatenate([[0], np.cumsum(n)]).astype(np.int32))
        q = queries(r, sum(n), 4, 128, "bf16").to(DEV)
        out = torch.empty_like(q)
        size = tq4.kv8_prefill_workspace_bytes(sum(n), 2, 4, 1, 128, 16, tables.shape[1], max(n))
        ws = torch.full((size,), 255, dtype=torch.uint8, device=DEV)
        assert size > 0
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            tq4.kv8_paged_prefill(q, kc, vc, sc, tables, L, cu, max(n), out=out, workspace=ws)
        for _ in range(3):
            q.copy_(queries(r, sum(n), 4, 128, "bf16"))
            out.zero_()
            g.replay()
            eager = tq4.kv8_paged_prefill(q, kc, vc, sc, tables, L, cu, max(n))
            torch.cuda.synchronize()
            assert torch.equal(out, eager)


def test_streams_and_devices(tq4):
    """Calls on a stream of their own, by argument and by context, two at once."""
    r = np.random.default_rng(22)
    lens = [2000, 700]
    c = cache(r, lens, 2, 16, 128, "int8")
    kc, vc, sc, tables = on_device(*c, "int8")
    L, q = dev(np.array(lens, np.int32)), queries(r, 2, 8, 128, "bf16").to(DEV)
    want = tq4.kv8_paged_decode(q, kc, vc, sc, tables, L)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for _ in range(10):
        outs.append(tq4.kv8_paged_decode(q, kc, vc, sc, tables, L, stream=a))
        with torch.cuda.stream(b):
            outs.append(tq4.kv8_paged_decode(q, kc, vc, sc, tables, L))
        outs.append(tq4.kv8_paged_decode(q, kc, vc, sc, tables, L))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
