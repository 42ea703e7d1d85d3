"""A model of windowed and whole layers: a table and a pool for each kind, planned twice a step from the same lengths.  The step
is the prefix that both plans serve; pages that one of them took beyond it stay named, none is lost."""
import numpy as np
import pytest

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


@pytest.mark.parametrize("B", [7, 80])
@pytest.mark.parametrize("window,sinks", [(100, 4), (1, 0), (200, 65)])
def test_two_plans_of_a_step(B, window, sinks):
    import torch
    rng = np.random.default_rng(B + window)
    i32 = dict(dtype=torch.int32, device="cuda")
    M, N = 24, 12 * B
    sizes = {0: 3 * B, window: 2 * B}  # (whole sequences soon run out of pages, windows now and then)
    kinds = {w: dict(table=torch.full((B, M), -1, **i32), ring=torch.from_numpy(rng.permutation(P).astype(np.int32)).cuda(),
                     state=torch.tensor([3, P], **i32), first=torch.zeros(B + 1, **i32)) for w, P in sizes.items()}
    n, shorter = np.zeros(B, np.int32), set()
    for step in range(60):
        new = np.where(rng.random(B) < 0.04, -1, rng.integers(0, 40, B)).astype(np.int32)
        new = np.where(n + new > M * ROWS - 3, -1, new).astype(np.int32)
        lens, more = torch.from_numpy(n).cuda(), torch.from_numpy(new).cuda()
        for w, k in kinds.items():
            tie_amd.KVPool(k["ring"], k["state"]).plan(k["table"], lens, more, k["table"], k["first"], n_tokens=N, window=w,
                                                       sinks=sinks if w else 0)
        whole, part = kinds[0]["first"], kinds[window]["first"]
        first = torch.minimum(whole, part)
        torch.cuda.synchronize()
        if not torch.equal(whole, part):
            shorter.add("whole" if int(whole[-1]) < int(part[-1]) else "windowed")
        first = first.cpu().numpy()
        got = np.diff(first)
        # a prefix of what is asked for
        asked = np.maximum(new, 0)
        served = int((np.cumsum(asked) <= first[-1]).sum())
        assert np.array_equal(got[:served], asked[:served]) and not got[served:].any(), step
        for w, P in sizes.items():
            table, ring, (head, free) = (kinds[w][x].cpu().numpy() for x in ("table", "ring", "state"))
            held = table[table >= 0].tolist()
            assert sorted(held + [int(ring[(head + i) % P]) for i in range(free)]) == list(range(P)), (step, w)
            for b in range(B):
                if new[b] < 0:
                    assert (table[b] == -1).all()
                    continue
                # what the step's tokens see and write is on pages
                see = [r for r in range(n[b] + got[b]) if w == 0 or r < sinks or r > n[b] - w] if got[b] else []
                assert all(table[b, r // ROWS] >= 0 for r in see), (step, w, b)
        n = np.where(new < 0, 0, n + got).astype(np.int32)
    assert shorter, "the plans never differed"
