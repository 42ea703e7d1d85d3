"""The page plan against the same written request by request; every array equal."""
import numpy as np
import pytest

import kv_ref
import tie_amd

pytestmark = pytest.mark.gpu
ROWS = 64


@pytest.fixture(scope="module", autouse=True)
def device():
    import torch
    assert torch.cuda.is_available(), "GPU test without a GPU"
    tie_amd.init(0)
    yield
    tie_amd.shutdown()


def expect(table, lens, new, ring, state, n_tokens, window, sinks):
    table, ring, M, P = table.copy(), ring.copy(), table.shape[1], len(ring)
    head, free = (int(x) for x in state)
    valid = 0 <= head < P and 0 <= free <= P
    if not valid:
        head = free = 0
    room = P - free if valid else 0
    pos, slot, first = np.full(n_tokens, -1, np.int32), np.full(n_tokens, -1, np.int32), [0]
    taken, back, stopped = 0, 0, False
    was = table.copy()
    for b in range(len(lens)):
        n, m = int(lens[b]), int(new[b])
        want = m if n >= 0 and m >= 0 and n + m <= M * ROWS else 0
        cols = [c for c in range(-(-n // ROWS), -(-(n + want) // ROWS)) if not 0 <= was[b, c] < P] if want else []
        if taken + len(cols) > free or first[-1] + want > n_tokens:
            stopped = True
        if stopped:
            first.append(first[-1])
        else:
            for c in cols:
                table[b, c] = ring[(head + taken) % P]
                taken += 1
            for j in range(want):
                t, r = first[-1] + j, n + j
                pos[t], page = r, table[b, r // ROWS]
                slot[t] = page * ROWS + r % ROWS if 0 <= page < P else -1
            first.append(first[-1] + want)
        if m < 0:
            gone = range(M)
        elif window:
            gone = [c for c in range(-(-sinks // ROWS), M) if (c + 1) * ROWS <= n - window + 1]
        else:
            gone = []
        for c in gone:
            if 0 <= was[b, c] < P and back < room:
                ring[(head + free + back) % P] = was[b, c]
                table[b, c] = -1
                back += 1
    after = [(head + taken) % P, free - taken + back] if valid else list(state)
    return table, np.array(first, np.int32), pos, slot, ring, np.array(after, np.int32)


def call(table, lens, new, ring, state, n_tokens, window=0, sinks=0, in_place=False, work=None):
    import torch
    cuda = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()  # noqa: E731
    table, lens, new, ring, state = (cuda(x) for x in (table, lens, new, ring, state))
    pool = tie_amd.KVPool(ring, state)
    out, state_out = (table, None) if in_place else (torch.full_like(table, -77), torch.full_like(state, -77))
    first = torch.full((len(lens) + 1,), -77, dtype=torch.int32, device="cuda")
    pos, slot = (torch.full((n_tokens + 2,), -77, dtype=torch.int32, device="cuda") for _ in range(2))
    keep = (table.clone(), state.clone())
    if work is not None:
        work = torch.zeros(tie_amd.kv_plan_work_bytes(len(lens)), dtype=torch.uint8, device="cuda")
    for _ in range(1 if in_place else 2):  # (again from the same state: the same)
        pool.plan(table, lens, new, out, first, pos=pos[:n_tokens], slot=slot[:n_tokens], state_out=state_out, window=window, sinks=sinks,
                  work=work)
    torch.cuda.synchronize()
    assert (pos[n_tokens:] == -77).all() and (slot[n_tokens:] == -77).all()
    if not in_place:
        assert torch.equal(table, keep[0]) and torch.equal(state, keep[1])
    return [x.cpu().numpy() for x in (out, first, pos[:n_tokens], slot[:n_tokens], ring, state if in_place else state_out)]


def requests(rng, B, M, free, long=False, holes=False):
    """Requests in the middle of a service, pages named once each."""
    lens = rng.integers(0, M * ROWS + 1, B) if long else np.minimum(rng.integers(0, 300, B), M * ROWS)
    new = rng.choice([0, 1, 1, 1, 5, 64, 65, 200, -1], B)
    held = -(-lens // ROWS) + rng.integers(0, 3, B)
    P = int(B * (M + 3) + free)
    ids = list(rng.permutation(P))
    table = np.full((B, M), -1, np.int32)
    for b in range(B):
        for c in range(min(M, held[b])):
            if not (holes and rng.random() < 0.3):
                table[b, c] = ids.pop()
    table[(table < 0) & (rng.random(table.shape) < 0.2)] = P + 5  # (a number that is no page)
    ring, head = np.full(P, -9, np.int32), int(rng.integers(P))
    for i in range(free):
        ring[(head + i) % P] = ids.pop()
    return table, lens.astype(np.int32), new.astype(np.int32), ring, np.array([head, free], np.int32)


def same(got, want):
    for name, a, b in zip(("table", "first", "pos", "slot", "ring", "state"), got, want):
        assert np.array_equal(a, b), (name, np.argwhere(a != b)[:5], a[a != b][:5], b[a != b][:5])


@pytest.mark.parametrize("B,M", [(1, 1), (1, 700), (2, 5), (5, 64), (15, 9), (16, 7), (17, 7), (63, 3), (64, 130), (65, 130), (200, 65), (1040, 6),
                                 (2500, 2)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (100, 4), (70, 64), (1 << 30, 1 << 30)])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan(B, M, window, sinks, in_place):
    rng = np.random.default_rng(B + window % 100)
    for free, rows, long, holes in ((B * 5 + 3, B * 250, True, False), (B * 5, B * 250, False, True), (B // 2, B * 20 + 1, False, False)):
        a = requests(rng, B, M, free, long, holes)
        same(call(*a, rows, window, sinks, in_place, work=True), expect(*a, rows, window, sinks))


@pytest.mark.parametrize("B", [3, 70, 1100])
def test_where_pages_or_rows_run_out(B):
    """At each place of the cut: none served, some, all but the last, just all; behind the cut requests that need nothing
    get nothing either."""
    rng = np.random.default_rng(B)
    table, lens, new, ring, _ = requests(rng, B, 8, 4 * B + 8)
    new = np.abs(new)
    need = [len([c for c in range(-(-n // ROWS), -(-(n + m) // ROWS)) if not 0 <= table[b, c] < len(ring)]) if n + m <= 8 * ROWS else 0
            for b, (n, m) in enumerate(zip(lens, new))]
    ring[:] = rng.permutation(len(ring))
    for free in sorted({0, 1, sum(need) // 2, max(0, sum(need) - 1), sum(need)}):
        state = np.array([len(ring) - 1, free], np.int32)
        same(call(table, lens, new, ring, state, 300 * B), expect(table, lens, new, ring, state, 300 * B, 0, 0))
    total = int(expect(table, lens, new, ring, np.array([3, len(ring)], np.int32), 300 * B, 0, 0)[1][-1])
    for rows in sorted({0, 1, total // 2, total - 1, total}):
        state = np.array([3, len(ring)], np.int32)
        same(call(table, lens, new, ring, state, rows), expect(table, lens, new, ring, state, rows, 0, 0))


@pytest.mark.parametrize("B", [2, 90])
def test_what_the_arrays_say_wrong(B):
    """Lengths below 0 or past the table, counts too large, rings that are none, ring entries that are no pages, and more
    pages back than the ring has places: nothing outside the arrays, and what the header says."""
    rng = np.random.default_rng(B)
    table, lens, new, ring, state = requests(rng, B, 6, 4 * B)
    lens[0], new[1] = -5, 0x7fffffff
    if B > 2:
        lens[5], lens[6], new[7], new[8] = 6 * ROWS + 1, 0x7fffffff, -0x80000000, 6 * ROWS + 1
    for window in (0, 40):
        same(call(table, lens, new, ring, state, 900, window), expect(table, lens, new, ring, state, 900, window, 0))
    P = len(ring)
    for bad in ([-1, 4], [P, 4], [0, P + 1], [3, -1], [0x7fffffff, 0x7fffffff], [-0x80000000, 1]):
        st = np.array(bad, np.int32)
        same(call(table, lens, new, ring, st, 900, 40), expect(table, lens, new, ring, st, 900, 40, 0))
    odd = ring.copy()
    odd[::2] = [P, -1, 0x7fffffff, -4][0]
    same(call(table, lens, new, odd, state, 900), expect(table, lens, new, odd, state, 900, 0, 0))
    ended, full = np.full(B, -1, np.int32), np.array([1, P - 1], np.int32)
    same(call(table, lens, ended, ring, full, 900), expect(table, lens, ended, ring, full, 900, 0, 0))


@pytest.mark.parametrize("n_tokens", [0, 7])
def test_no_requests(n_tokens):
    none = np.zeros(0, np.int32)
    ring, state = np.arange(9, dtype=np.int32), np.array([4, 5], np.int32)
    table = np.zeros((0, 3), np.int32)
    same(call(table, none, none, ring, state, n_tokens), expect(table, none, none, ring, state, n_tokens, 0, 0))


def test_long_prompts():
    """Prompts of several chunks of 4096 rows, with and without pages that the table names already."""
    rng = np.random.default_rng(0)
    M, P = 600, 6000
    ids = rng.permutation(P).astype(np.int32)
    table = np.full((6, M), -1, np.int32)
    lens, new = np.array([0, 100, 64, 3000, 9, 0], np.int32), np.array([20000, 9001, 1, 15000, 30000, 0], np.int32)
    table[1, :2], table[2, :1], table[3, :47], table[4, :1] = ids[:2], ids[2:3], ids[3:50], ids[50:51]
    table[3, 100:103], table[4, 300] = ids[51:54], ids[54]  # (named ahead of their rows)
    ring = np.zeros(P, np.int32)
    ring[np.arange(P - 55)] = ids[55:]
    state = np.array([0, P - 55], np.int32)
    for rows in (80000, 60000, 16000):
        same(call(table, lens, new, ring, state, rows), expect(table, lens, new, ring, state, rows, 0, 0))


def test_no_page_is_lost_or_given_twice():
    """A service over a hundred steps in one graph: every page in the pool or in one row of the table, always."""
    import torch
    rng = np.random.default_rng(1)
    B, M, P, N, window = 40, 30, 500, 400, 300
    i32 = dict(dtype=torch.int32, device="cuda")
    table, lens, new, first = torch.full((B, M), -1, **i32), torch.zeros(B, **i32), torch.zeros(B, **i32), torch.zeros(B + 1, **i32)
    ring, state = torch.from_numpy(rng.permutation(P).astype(np.int32)).cuda(), torch.tensor([17, P], **i32)
    pool, graph, pos = tie_amd.KVPool(ring, state), torch.cuda.CUDAGraph(), torch.zeros(N, **i32)
    work = torch.zeros(tie_amd.kv_plan_work_bytes(B), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    with kv_ref.capture(graph):
        pool.plan(table, lens, new, table, first, pos=pos, window=window, sinks=4, work=work)
    want = [x.cpu().numpy() for x in (table, ring, state)]
    n = np.zeros(B, np.int32)
    for step in range(100):
        m = np.where(rng.random(B) < 0.03, -1, np.where(n == 0, rng.integers(0, 150, B), rng.integers(0, 3, B))).astype(np.int32)
        m = np.where(n + m > M * ROWS - 5, -1, m).astype(np.int32)
        lens.copy_(torch.from_numpy(n))
        new.copy_(torch.from_numpy(m))
        graph.replay()
        torch.cuda.synchronize()
        want_t, want_f, want_p, _, want_r, want_s = expect(want[0], n, m, want[1], want[2], N, window, 4)
        got = [x.cpu().numpy() for x in (table, first, pos, ring, state)]
        for a, b in zip(got, (want_t, want_f, want_p, want_r, want_s)):
            assert np.array_equal(a, b), step
        want = [want_t, want_r, want_s]
        held = want_t[want_t >= 0].tolist()
        free = [int(want_r[(want_s[0] + i) % P]) for i in range(want_s[1])]
        assert sorted(held + free) == list(range(P)), step
        n = np.where(m < 0, 0, n + np.diff(want_f)).astype(np.int32)


def test_sums_that_pass_32_bits():
    """Requests that ask for 2^26 rows each, 70 of them: nothing fits, or what stands before them."""
    import torch
    i32 = dict(dtype=torch.int32, device="cuda")
    B, M = 70, 1 << 20
    table, lens, new = torch.full((B, M), -1, **i32), torch.zeros(B, **i32), torch.full((B,), 1 << 26, **i32)
    ring, state = torch.arange(50, **i32), torch.tensor([48, 50], **i32)
    pool, first, pos = tie_amd.KVPool(ring, state), torch.zeros(B + 1, **i32), torch.zeros(100, **i32)
    after = torch.zeros(2, **i32)
    for small in (0, 3):
        new[:small] = 30
        pool.plan(table, lens, new, table, first, pos=pos, state_out=after)
        torch.cuda.synchronize()
        assert first.tolist() == [30 * min(b, small) for b in range(B + 1)]
        assert after.tolist() == [(48 + small) % 50, 50 - small]
        assert pos.tolist() == list(range(30)) * small + [-1] * (100 - 30 * small)
    assert table[:4, 0].tolist() == [48, 49, 0, -1] and (table[:, 1:] == -1).all()
    # as many token rows as an int names: the first request does not lie within its row of the table, the second (64
    # rows) and the third (30) have their pages already, and the fourth wants more than there are
    new[:2] = torch.tensor([0x7fffffff - 63, 64], **i32)
    pool.plan(table, lens, new, table, first, n_tokens=0x7fffffff, state_out=after)
    torch.cuda.synchronize()
    assert first.tolist() == [0, 0, 64] + [94] * (B - 2)
    assert after.tolist() == [48, 50]
