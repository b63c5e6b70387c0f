"""tq4_paged_plan against the plan request by request: every output, the tables
and the ring whole."""
import numpy as np
import pytest
import torch

import kv8_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def case(seed, B, S, M, new_hi=1, spare=1.0, leave=0.0, extra_room=5, odd=False):
    """A batch whose tables hold distinct pages, and the pool's other pages free."""
    r = np.random.default_rng(seed)
    ctx = r.integers(0, M * S + 1, B)
    new = r.integers(0, new_hi + 1, B)
    ctx = np.where(r.random(B) < 0.8, np.minimum(ctx, M * S - new), ctx)
    ctx = np.maximum(ctx, 0)
    ctx[r.random(B) < 0.2] //= S * S  # page borders and empty ones
    release = (r.random(B) < leave).astype(np.int32)
    held = -(-ctx // S)
    want = np.maximum(-(-(np.where(release, 0, ctx) + new) // S) - np.where(release, 0, held), 0)
    free = max(1, int(spare * want.sum()))
    P = int(held.sum()) + free
    order = r.permutation(P).astype(np.int32)
    tables = np.full((B, M), -7, np.int32)
    at = 0
    for b in range(B):
        tables[b, :held[b]] = order[at:at + held[b]]
        at += held[b]
    ring, head = np.full(P, -9, np.int32), int(r.integers(0, P))
    ring[(head + np.arange(free)) % P] = order[at:]
    ctx = ctx.astype(np.int32)
    new = new.astype(np.int32)
    if odd:  # lengths and entries that no caller should pass
        ctx[r.integers(0, B)] = -5
        ctx[r.integers(0, B)] = M * S + 100
        new[r.integers(0, B)] = -3
        tables[r.integers(0, B), 0] = P + 4
        tables[r.integers(0, B), 0] = -1
    room = int(np.maximum(new, 0).sum()) + extra_room
    return dict(ctx=ctx, new=new, release=release, tables=tables, ring=ring,
                state=np.array([head, free], np.int32), S=S, room=max(room, 0))


def run(tq4, c, release=True, positions=True, in_place=False):
    d = {k: torch.from_numpy(np.ascontiguousarray(c[k])).to(DEV)
         for k in ("ctx", "new", "release", "tables", "ring", "state")}
    B = len(c["ctx"])
    e = lambda n: torch.full((n,), -77, dtype=torch.int32, device=DEV)  # noqa: E731
    o = dict(slots=e(c["room"]), positions=e(c["room"]) if positions else None, cu=e(B + 1),
             granted=e(B), lens=None if in_place else e(B), state=None if in_place else e(2))
    print("plan", B, c["S"], c["tables"].shape, c["room"], flush=True)
    tq4.paged_plan(d["ctx"], d["new"], d["tables"], d["ring"], d["state"], o["slots"], o["cu"],
                   o["granted"], c["S"], release=d["release"] if release else None,
                   positions=o["positions"], new_context_lens=o["lens"],
                   new_free_state=o["state"])
    torch.cuda.synchronize()
    if in_place:
        o["lens"], o["state"] = d["ctx"], d["state"]
    o["tables"], o["ring"] = d["tables"], d["ring"]
    return {k: None if v is None else v.cpu().numpy() for k, v in o.items()}


def same(got, c, release=True):
    want = ref.plan(c["ctx"], c["new"], c["release"] if release else None, c["tables"], c["ring"],
                    c["state"], c["S"], c["room"])
    for k, w in want.items():
        if got[k] is not None:
            assert np.array_equal(got[k], w), (k, np.argwhere(got[k] != w)[:5].tolist())


CASES = [
    # B, S, M, new_hi, spare, leave, extra_room, odd
    (1, 16, 4, 1, 1.0, 0.0, 0, False),
    (1, 16, 9, 100, 1.0, 0.0, 7, False),
    (2, 48, 5, 3, 0.5, 0.5, 1, False),
    (63, 16, 33, 1, 1.0, 0.0, 1, False),
    (64, 16, 512, 1, 1.0, 0.0, 0, False),
    (65, 32, 17, 70, 1.0, 0.2, 3, False),
    (257, 16, 20, 40, 0.6, 0.3, 64, False),
    (1025, 128, 6, 300, 0.7, 0.1, -9, False),   # rows that do not fit the map
    (3000, 16, 7, 2, 0.9, 0.3, 33, False),
    (40, 16, 6, 30, 0.8, 0.3, 2, True),
    (900, 32, 8, 90, 0.5, 0.4, -100, True),
]


@pytest.mark.parametrize("k", range(len(CASES)))
def test_plan(tq4, k):
    c = case(k, *CASES[k])
    same(run(tq4, c), c)


@pytest.mark.parametrize("k", range(0, len(CASES), 2))
def test_plan_in_place_and_without_options(tq4, k):
    c = case(100 + k, *CASES[k])
    same(run(tq4, c, in_place=True), c)
    same(run(tq4, c, release=False, positions=False), c, release=False)


def test_plan_no_rows_and_no_free_pages(tq4):
    c = case(7, 5, 16, 4, 0)
    c["room"] = 0
    same(run(tq4, c), c)
    c = case(8, 50, 16, 4, 40)
    c["state"][1] = 0
    same(run(tq4, c), c)
    c["state"][:] = (-3, 10 ** 6)  # a state that no caller should pass
    same(run(tq4, c), c)


def test_plan_lengths_past_32_bits(tq4):
    """Rows that pass 2^31 are refused and cu_seqlens saturates."""
    c = case(9, 6, 16, 4, 8)
    c["new"][:] = 2 ** 31 - 1
    c["new"][1] = 3
    c["room"] = 64
    same(run(tq4, c), c)


def test_plan_steps_drive_a_pool(tq4):
    """Steps in a row, in place: no page is held twice or lost."""
    r = np.random.default_rng(3)
    B, S, M, P = 37, 16, 12, 200
    tables = np.full((B, M), -1, np.int32)
    c = dict(ctx=np.zeros(B, np.int32), tables=tables, ring=r.permutation(P).astype(np.int32),
             state=np.array([190, P], np.int32), S=S)
    for step in range(25):
        c["new"] = r.integers(0, 40 if step % 5 == 0 else 2, B).astype(np.int32)
        c["release"] = (r.random(B) < 0.1).astype(np.int32)
        c["room"] = int(c["new"].sum()) + 3
        got = run(tq4, c, in_place=True)
        same(got, c)
        c.update(ctx=got["lens"], tables=got["tables"], ring=got["ring"], state=got["state"])
        head, count = c["state"]
        free = c["ring"][(head + np.arange(count)) % P]
        held = np.concatenate([c["tables"][b, :-(-c["ctx"][b] // S)] for b in range(B)])
        assert len(np.unique(np.concatenate([free, held]))) == P == count + len(held)


def test_plan_captured(tq4):
    """A captured plan, replayed with eager work between, step after step."""
    c = case(21, 33, 16, 64, 2)
    d = {k: torch.from_numpy(c[k]).to(DEV) for k in ("ctx", "new", "release", "tables", "ring", "state")}
    e = lambda n: torch.zeros(n, dtype=torch.int32, device=DEV)  # noqa: E731
    slots, cu, granted = e(c["room"]), e(34), e(33)
    ws = torch.empty(1 << 16, dtype=torch.uint8, device=DEV)
    start = {k: v.clone() for k, v in d.items()}
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        tq4.paged_plan(d["ctx"], d["new"], d["tables"], d["ring"], d["state"], slots, cu, granted,
                       16, release=d["release"], workspace=ws)
    for k in d:
        d[k].copy_(start[k])
    for _ in range(3):
        want = ref.plan(c["ctx"], c["new"], c["release"], c["tables"], c["ring"], c["state"], 16,
                        c["room"])
        g.replay()
        torch.cuda.synchronize()
        assert np.array_equal(slots.cpu().numpy(), want["slots"])
        assert np.array_equal(d["tables"].cpu().numpy(), want["tables"])
        assert np.array_equal(d["state"].cpu().numpy(), want["state"])
        c.update(ctx=want["lens"].astype(np.int32), tables=want["tables"], ring=want["ring"],
                 state=want["state"].astype(np.int32))
        torch.ones(1000, device=DEV).sum().item()
