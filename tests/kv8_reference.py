"""The 8-bit paged cache's operators by definition (numpy, 64 bits), for the
tests of include/tq4_kv8.h."""
import numpy as np
import torch

CODE_MAX = {"fp8": 448.0, "int8": 127.0}
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
CODES = {"fp8": torch.float8_e4m3fn, "int8": torch.int8}
LEAST, MOST = 2.0 ** -100, 2.0 ** 120


def fp8_values():
    """What the 256 bytes of OCP e4m3 stand for."""
    t = np.empty(256)
    for b in range(256):
        e, f = (b >> 3) & 15, b & 7
        x = f * 2.0 ** -9 if e == 0 else (8 + f) * 2.0 ** (e - 10)
        t[b] = np.nan if (b & 127) == 127 else -x if b & 128 else x
    return t


FP8 = fp8_values()


def code_values(raw, code):
    """Bytes (uint8) as the numbers they stand for."""
    return FP8[raw] if code == "fp8" else raw.view(np.int8).astype(np.float64)


def to_codes(x, code):
    """FP32 values as bytes: nearest, ties to even, saturated; NaN the largest."""
    x = np.where(np.isnan(x), np.inf, np.asarray(x, np.float64))
    x = np.clip(x, -CODE_MAX[code], CODE_MAX[code])
    if code == "int8":
        return np.rint(x).astype(np.int8).view(np.uint8)
    grid = FP8[:127]
    a = np.abs(x)
    hi = np.minimum(np.searchsorted(grid, a), 126)
    lo = np.maximum(hi - 1, 0)
    up, down = grid[hi] - a, a - grid[lo]
    pick = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    return (pick | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


# ------------------------------------------------------------------- the plan
def plan(ctx, new, release, tables, ring, state, S, room):
    """The plan, request by request. Copies; returns a dict of every output."""
    tables, ring = tables.copy(), ring.copy()
    B, M = tables.shape
    P = len(ring)
    old_ring, old_tables = ring.copy(), tables.copy()
    head, count = int(state[0]) % P, min(max(int(state[1]), 0), P)
    cap = min(M * S, 2 ** 31 - 1)
    cu, granted, lens = [0], [], []
    slots, pos = np.full(room, -1, np.int64), np.zeros(room, np.int64)
    total = wanted = taken = backs = 0
    for b in range(B):
        c, n = min(max(int(ctx[b]), 0), cap), max(int(new[b]), 0)
        first = total
        total += n
        cu.append(min(total, 2 ** 31 - 1))
        if release is not None and release[b]:
            for i in range(-(-c // S)):
                if count + backs < P:
                    ring[(head + count + backs) % P] = old_tables[b, i]
                backs += 1
            c = 0
        held, want = -(-c // S), -(-(c + n) // S) - -(-c // S)
        ok = c + n <= cap and total <= room
        if ok:
            wanted += want
            ok = want == 0 or wanted <= count
        if ok:
            for i in range(want):
                tables[b, held + i] = old_ring[(head + wanted - want + i) % P]
            taken += want
            for t in range(n):
                page = int(tables[b, (c + t) // S])
                pos[first + t] = c + t
                if 0 <= page < P:
                    slots[first + t] = page * S + (c + t) % S
        granted.append(n if ok else 0)
        lens.append(c + n if ok else c)
    return dict(tables=tables, ring=ring, slots=slots, positions=pos, cu=np.array(cu),
                granted=np.array(granted), lens=np.array(lens),
                state=np.array([(head + taken) % P, min(P, count - taken + backs)]))


# ----------------------------------------------------------------- the writer
def need_scale(amax, code):
    s = LEAST
    while amax > CODE_MAX[code] * s:
        s *= 2.0
    return s


def write(key, value, kc, vc, sc, slots, code):
    """Rows of key and value (FP32 arrays holding the activations' values) into
    copies of the byte pools kc [P][H][S][d], vc [P][H][S/16][d][16] and the
    scales [2][P][H]."""
    kc, vc, sc = kc.copy(), vc.copy(), sc.copy()
    P, H, S, d = kc.shape
    row_of = {int(s): t for t, s in enumerate(slots) if 0 <= s < P * S}  # the later one
    rows_of = {}
    for s, t in row_of.items():
        rows_of.setdefault(s // S, []).append(t)
    # the value pool with tokens before channels
    vt = np.ascontiguousarray(vc.transpose(0, 1, 2, 4, 3)).reshape(P, H, S, d)
    for page, rows in rows_of.items():
        opened = any(slots[t] % S == 0 for t in rows)
        for plane, x, pool in ((0, key, kc), (1, value, vt)):
            for h in range(H):
                a = np.abs(x[rows, h])
                a = a[np.isfinite(a)]
                need = need_scale(float(a.max()) if a.size else 0.0, code)
                was = np.float32(sc[plane, page, h])
                old = was if not opened and was > 0 and np.isfinite(was) else np.float32(0)
                now = np.float32(max(float(old), need))
                if not opened and old < now:
                    held = code_values(pool[page, h], code).astype(np.float32)
                    nan = np.isnan(held)
                    moved = to_codes(held * np.float32(old / now), code)
                    pool[page, h] = np.where(nan, pool[page, h], moved)
                for t in rows:
                    with np.errstate(over="ignore", invalid="ignore"):
                        pool[page, h, slots[t] % S] = to_codes(
                            x[t, h] * (np.float32(1) / now), code)
                sc[plane, page, h] = now
    vc = np.ascontiguousarray(vt.reshape(P, H, S // 16, 16, d).transpose(0, 1, 2, 4, 3))
    return kc, vc, sc


# -------------------------------------------------------------- the attention
def attention(q, kc, vc, sc, tables, lens, cu, code, causal, scale, max_q=None):
    """out and, element by element, what an implementation may be off it.

    q [rows][Hq][d] float64, the caches as bytes. The bound counts, in units of
    A = sum p |v| / sum p (the row's weighted magnitude):
      - a weight rounded to FP16: 2^-11 relative, 2^-25 absolute where it is
        subnormal (the row's largest product being at least 2^6: 2^-31 of it);
      - an error e of the exponent changes a weight by e relative, the sum of
        weights too: 2 e. e: d products accumulated in FP32 (d 2^-24 of sum
        |q k|), the FP16 operand's subnormals (2^-25 of the row's largest |q|
        an element, times |k|), and 8 roundings of the exponent's magnitude;
      - the FP32 sums over n tokens and the merges: (n + 64) 2^-24.
    The caller adds the output's own rounding."""
    rows, Hq, d = q.shape
    P, H, S, _ = kc.shape
    G = Hq // H
    vt = vc.transpose(0, 1, 2, 4, 3).reshape(P, H, S, d)
    out, off = np.zeros((rows, Hq, d)), np.zeros((rows, Hq, d))
    done = np.zeros(rows, bool)
    scales = np.clip(sc.astype(np.float64), LEAST, MOST)
    for b in range(len(lens)):
        n = min(max(int(lens[b]), 0), tables.shape[1] * S)
        r0, r1 = int(cu[b]), int(cu[b + 1])
        at = np.arange(n)
        page = tables[b][at // S]
        fine = (page >= 0) & (page < P)
        at, page = at[fine], page[fine]
        for h in range(H):
            k = code_values(kc[page, h, at % S], code) * scales[0, page, h][:, None]
            v = code_values(vt[page, h, at % S], code) * scales[1, page, h][:, None]
            for r in range(r0, r1 if max_q is None else min(r1, r0 + max_q)):
                done[r] = True
                see = at <= n - (r1 - r0) + (r - r0) if causal else np.ones(len(at), bool)
                if not see.any():
                    continue
                ks, vs = k[see], v[see]
                for g in range(h * G, h * G + G):
                    x = q[r, g]
                    s = scale * (ks @ x)
                    size = np.abs(scale) * (np.abs(ks) @ np.abs(x))
                    e = (d * 2.0 ** -24 * size +
                         2.0 ** -25 * np.abs(x).max() * np.abs(scale) * np.abs(ks).sum(1) +
                         8 * 2.0 ** -24 * (np.abs(s) + 128)).max()
                    p = np.exp(s - s.max())
                    A = (p[:, None] * np.abs(vs)).sum(0) / p.sum()
                    big = (p[:, None] * np.abs(vs)).max() / p.sum()
                    out[r, g] = (p[:, None] * vs).sum(0) / p.sum()
                    off[r, g] = (A * (2.0 ** -11 + 2 * e + (len(ks) + 64) * 2.0 ** -24) +
                                 len(ks) * 2.0 ** -31 * big * 448)
    return out, off, done


def check(got, want, off, dtype):
    """got (a torch tensor) within `off` and its own rounding of want."""
    half = torch.finfo(dtype).eps / 2
    g = got.double().cpu().numpy()
    tiny = torch.finfo(dtype).tiny * half * 2
    bound = off + half * (np.abs(want) + off) + tiny
    bad = ~(np.abs(g - want) <= bound)
    assert not bad.any(), (f"{bad.sum()} of {bad.size} off; worst "
                           f"{np.nanmax(np.abs(g - want) / bound):.3g} of the bound, first at "
                           f"{np.argwhere(bad)[0].tolist()}: {g[bad][0]} for {want[bad][0]}")
    return float(np.max(np.abs(g - want) / bound)) if g.size else 0.0
