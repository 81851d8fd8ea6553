"""GPU tests of PagePool.fork on pairs that it must not make: the target, the counts and the tails stay as they are,
the status says why, and the other pairs of the call go through."""

import pytest
import torch

import nvfp4_attn_kernel_b200._lib as L
from nvfp4_attn_kernel_b200.nvfp4_vllm.pages import PagePool

pytestmark = pytest.mark.gpu

ROWS, COLUMNS, PAGES, LAYERS, SLOTS = 6, 5, 30, 3, 8
NAMES = ("table", "held", "full", "used", "refs", "tail_key", "tail_value")


def ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


class Rows:
    """Rows 0 to 2 hold three pages each and a tail, rows 3 to 5 nothing; a fork of 0 to 3 and of 1 to 4."""

    def __init__(self, device, heads):
        g = torch.Generator().manual_seed(heads)
        self.table = torch.full((ROWS, COLUMNS), -1, dtype=torch.int32)
        self.table[:3, :3] = torch.randperm(PAGES - 1, generator=g)[:9].int().view(3, 3) + 1
        refs = torch.zeros(PAGES, dtype=torch.int32)
        refs[self.table[:3, :3].flatten().long()] = 1
        self.table, self.refs = self.table.to(device), refs.to(device)
        self.held, self.full = ints([3, 3, 3, 0, 0, 0], device), ints([384, 384, 384, 0, 0, 0], device)
        self.used, self.slots = ints([100, 128, 7, 0, 0, 0], device), ints([4, 1, 0, 7, 2, 5], device)
        self.tail_key, self.tail_value = (torch.randn(LAYERS, SLOTS, 128, heads, 128, generator=g).to(torch.bfloat16).to(device)
                                          for _ in range(2))
        self.pool = PagePool([torch.zeros(PAGES, 64, dtype=torch.uint8, device=device)], refs=self.refs, tail_key=self.tail_key,
                             tail_value=self.tail_value, reserved_pages=1)
        self.sources, self.targets = ints([0, 1], device), ints([3, 4], device)

    def state(self):
        return {name: getattr(self, name).clone() for name in NAMES}

    def fork(self, sources=None, targets=None):
        self.pool.fork(self.sources if sources is None else sources, self.targets if targets is None else targets, self.table,
                       self.held, self.full, self.used, self.slots)


CHANGES = [
    ("held", 3, 2, L.STATUS_BAD_ROW), ("held", 3, -1, L.STATUS_BAD_ROW),                 # the target holds pages
    ("held", 0, -1, L.STATUS_BAD_LENGTH), ("held", 0, COLUMNS + 1, L.STATUS_BAD_LENGTH),
    ("full", 0, 200, L.STATUS_BAD_LENGTH), ("full", 0, -128, L.STATUS_BAD_LENGTH),
    ("used", 0, -1, L.STATUS_BAD_LENGTH), ("used", 0, 129, L.STATUS_BAD_LENGTH),
    ("slots", 0, -1, L.STATUS_BAD_TAIL_ID), ("slots", 0, SLOTS, L.STATUS_BAD_TAIL_ID),
    ("slots", 3, -1, L.STATUS_BAD_TAIL_ID), ("slots", 3, 1 << 30, L.STATUS_BAD_TAIL_ID),
    ("slots", 3, 4, L.STATUS_BAD_TAIL_ID),                                               # the source's own slot
    ("slots", 3, 1, L.STATUS_BAD_TAIL_ID),                                               # the other pair's source's
    ("table", (0, 2), -1, L.STATUS_BAD_PAGE_ID), ("table", (0, 0), PAGES, L.STATUS_BAD_PAGE_ID),
]


@pytest.mark.parametrize("heads", [1, 8])
@pytest.mark.parametrize("name,at,value,bit", CHANGES)
def test_a_refused_pair_changes_nothing(cuda_device, heads, name, at, value, bit):
    rows = Rows(cuda_device, heads)
    getattr(rows, name)[at] = value
    want = rows.state()
    rows.fork()
    assert int(rows.pool.status) == bit
    # the other pair, by hand
    want["table"][4, :3] = want["table"][1, :3]
    want["refs"][want["table"][1, :3].long()] += 1
    want["held"][4], want["full"][4], want["used"][4] = 3, 384, 128
    for x in (want["tail_key"], want["tail_value"]):
        x[:, 2] = x[:, 1]
    for key in NAMES:
        assert torch.equal(getattr(rows, key), want[key]), key


def test_targets_that_share_a_slot(cuda_device):
    rows = Rows(cuda_device, 2)
    rows.slots[4] = rows.slots[3]
    want = rows.state()
    rows.fork()
    assert int(rows.pool.status) == L.STATUS_BAD_TAIL_ID
    assert all(torch.equal(getattr(rows, key), want[key]) for key in NAMES)


@pytest.mark.parametrize("held", [0, 1, 2])
def test_a_source_that_holds_less_gives_a_whole_prefix(cuda_device, held):
    """Pages that the source's length names but that it does not hold: what it holds is shared, and the tail, which would
    come after them, is not: the target's history has no hole."""
    rows = Rows(cuda_device, 2)
    rows.held[0] = held
    rows.used[3] = 55
    tails = rows.tail_key.clone()
    rows.fork(rows.sources[:1], rows.targets[:1])
    assert int(rows.pool.status) == L.STATUS_BAD_LENGTH
    assert (int(rows.held[3]), int(rows.full[3]), int(rows.used[3])) == (held, held * 128, 0)
    assert torch.equal(rows.table[3, :held], rows.table[0, :held]) and torch.equal(rows.tail_key, tails)
    assert rows.refs[rows.table[0, :3].long()].tolist() == [2] * held + [1] * (3 - held)


def test_a_slot_does_not_matter_without_a_tail(cuda_device):
    rows = Rows(cuda_device, 2)
    rows.used[0], rows.slots[3] = 0, -1
    rows.fork()
    assert int(rows.pool.status) == 0 and rows.held.tolist() == [3, 3, 3, 3, 3, 0] and rows.used.tolist() == [0, 128, 7, 0, 128, 0]


def test_refused_and_healthy_replays(cuda_device):
    """One captured fork: refused while the target holds pages, made once they are released, refused again after."""
    rows = Rows(cuda_device, 1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rows.fork()
    for expect in (0, L.STATUS_BAD_ROW, L.STATUS_BAD_ROW):
        before = rows.state()
        graph.replay()
        torch.cuda.synchronize()
        assert int(rows.pool.status) == expect
        if expect:
            assert all(torch.equal(getattr(rows, key), before[key]) for key in NAMES)
    rows.pool.release(rows.targets, rows.table, rows.held)
    rows.pool.status.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert int(rows.pool.status) == 0 and rows.held.tolist() == [3, 3, 3, 3, 3, 0]
