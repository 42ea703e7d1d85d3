"""The page plan where sixteen requests' counts together pass 32 bits: what stands before them keeps its rows."""
import numpy as np
import pytest

import tie_amd

pytestmark = pytest.mark.gpu
PAGES = 1 << 22  # columns: a request of all their rows asks for 2^28


@pytest.fixture(scope="module", autouse=True)
def device():
    import torch
    assert torch.cuda.is_available(), "GPU test without a GPU"
    tie_amd.init(0)
    yield
    tie_amd.shutdown()


def expect(new, n_tokens, free):
    """first, and the pages taken, of requests that begin: a page for each 64 rows."""
    first, taken, stopped = [0], 0, False
    for m in new:
        need = -(-m // 64)
        stopped = stopped or first[-1] + m > n_tokens or taken + need > free
        first.append(first[-1] + (0 if stopped else m))
        taken += 0 if stopped else need
    return first, taken


# (sixteen of 2^28 sum to 2^32, with one 64 rows shorter to 2^32 - 64; the served ones before them to 100.  In the last case
# the first of the large ones' block is served too)
@pytest.mark.parametrize("before,after", [(16, 16), (16, 1), (32, 0), (17, 15)])
@pytest.mark.parametrize("short", [0, 64])
@pytest.mark.parametrize("n_tokens", [130, 0x7fffffff])
def test_a_block_of_requests_whose_sum_passes_32_bits(before, after, short, n_tokens):
    import torch
    i32 = dict(dtype=torch.int32, device="cuda")
    new = [100 // before] * (before - 1)
    new = new + [100 - sum(new)] + [(1 << 28) - short] + [1 << 28] * 15 + [3] * after
    B, free = len(new), 64
    if B <= 64:  # (more requests than one workgroup takes)
        new, B = new + [2] * (65 - B), 65
    table, lens = torch.full((B, PAGES), -1, **i32), torch.zeros(B, **i32)
    ring, state, after_state = torch.arange(free, **i32), torch.tensor([60, free], **i32), torch.zeros(2, **i32)
    first = torch.full((B + 1,), -77, **i32)
    sized = n_tokens < 1000
    pos, slot = (torch.full((n_tokens,), -77, **i32) if sized else None for _ in range(2))
    work = torch.zeros(tie_amd.kv_plan_work_bytes(B), dtype=torch.uint8, device="cuda")
    tie_amd.KVPool(ring, state).plan(table, lens, torch.tensor(new, **i32), table, first, pos=pos, slot=slot, n_tokens=n_tokens,
                                     state_out=after_state, work=work)
    torch.cuda.synchronize()
    want, taken = expect(new, n_tokens, free)
    assert want[-1] == 100 and first.tolist() == want
    assert after_state.tolist() == [(60 + taken) % free, free - taken]
    rows = [j for m in new[:before] for j in range(m)]
    pages = [(60 + b) % free for b, m in enumerate(new[:before]) for _ in range(m)]  # (each a page: 3 to 55 rows)
    if sized:
        assert pos.tolist() == rows + [-1] * (n_tokens - 100)
        assert slot.tolist() == [p * 64 + j for p, j in zip(pages, rows)] + [-1] * (n_tokens - 100)
    assert table[:before, 0].tolist() == [(60 + b) % free for b in range(before)]
    assert (table[:before, 1:] == -1).all() and (table[before:] == -1).all()


def test_a_block_of_large_requests_far_behind():
    """Cuts before and in the sixty-sixth block of requests, among counts of nearly 2^31 that no row of the table holds
    (those ask for nothing)."""
    import torch
    i32 = dict(dtype=torch.int32, device="cuda")
    B, M = 1200, 40
    rng = np.random.default_rng(0)
    new = rng.integers(0, 3, B)
    new[1040:1056] = M * 64
    new[::7] = 0x7fffffff
    for n_tokens in (1500, 20000):
        want = [0]
        stopped = False
        for m in np.where(new > M * 64, 0, new).tolist():
            stopped = stopped or want[-1] + m > n_tokens
            want.append(want[-1] + (0 if stopped else m))
        table, lens = torch.full((B, M), -1, **i32), torch.zeros(B, **i32)
        ring, state, first = torch.arange(3000, **i32), torch.tensor([0, 3000], **i32), torch.zeros(B + 1, **i32)
        pos = torch.full((n_tokens,), -77, **i32)
        tie_amd.KVPool(ring, state).plan(table, lens, torch.from_numpy(new.astype(np.int32)).cuda(), table, first, pos=pos)
        torch.cuda.synchronize()
        assert first.tolist() == want
        assert (pos[: want[-1]] >= 0).all() and (pos[want[-1]:] == -1).all()
