"""Pages copied, forked, freed, reserved and compacted on the device, against the
plain Python table (exact: these are whole numbers and moved bits)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from _ops64 import Pages
from llm_serving_runtime_b200 import DevicePages, copy_pages

pytestmark = pytest.mark.gpu


def _caches(P, g, kinds=("bf16", "scale")):
    out = []
    for kind in kinds:
        if kind == "bf16":
            out.append(torch.randn(P, 2, 3, 16, 64, generator=g, device="cuda").to(torch.bfloat16))
        elif kind == "fp8":
            out.append(torch.randint(0, 120, (P, 2, 8, 48), generator=g, device="cuda").to(torch.uint8))
        elif kind == "scale":
            out.append(torch.rand(P, 5, generator=g, device="cuda"))
        elif kind == "odd":
            out.append(torch.randint(0, 255, (P, 37), generator=g, device="cuda").to(torch.uint8))
        elif kind == "layer":  # one layer of a pool: page stride larger than the page
            out.append(torch.randn(P, 4, 2, 16, 64, generator=g, device="cuda").to(torch.float16)[:, 1])
        elif kind == "strided":  # segments: every other row
            out.append(torch.randn(P, 12, 64, generator=g, device="cuda")[:, ::2])
    return out


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("kinds", [("bf16", "scale"), ("layer", "strided", "fp8"), ("odd",), ("scale", "odd", "bf16")])
@pytest.mark.parametrize("P,n", [(2, 1), (50, 20), (400, 199)])
def test_copy_pages(kinds, P, n):
    g = _gen(P + n)
    caches = _caches(P, g, kinds)
    ids = torch.randperm(P, generator=g, device="cuda").to(torch.int32)
    src, dst = ids[:n].clone(), ids[n: 2 * n].clone()
    src[n // 2] = -1 if n > 1 else src[0]
    want = [c.clone() for c in caches]
    for w, c in zip(want, caches):
        on = src >= 0
        w[dst[on].long()] = c[src[on].long()]
    copy_pages(caches, src, dst, validate=True)
    for w, c in zip(want, caches):
        assert torch.equal(w, c)


def test_copy_pages_of_many_layers_and_large_pages():
    g = _gen(1)
    a = torch.randn(30, 40, 8, 16, 128, generator=g, device="cuda").to(torch.bfloat16)  # 1.3 MB a page
    b = a.flip(0).contiguous()
    wa, wb = a.clone(), b.clone()
    src, dst = _i32([3, 29, 7]), _i32([0, 1, 28])
    wa[dst.long()], wb[dst.long()] = a[src.long()], b[src.long()]
    copy_pages([a, b], src, dst, validate=True)
    assert torch.equal(a, wa) and torch.equal(b, wb)


def test_copy_pages_interleaved_by_layer():
    """A pool stored layer by layer, its pages [block, layer, ...] as a strided view."""
    g = torch.Generator().manual_seed(21)
    pool = torch.randn(5, 40, 3, 16, 64, generator=g).cuda()
    want = pool.clone()
    want[:, [7, 39]] = want[:, [0, 12]]
    copy_pages([pool.transpose(0, 1)], torch.tensor([0, 12], dtype=torch.int32).cuda(),
               torch.tensor([7, 39], dtype=torch.int32).cuda())
    assert torch.equal(pool, want)


def test_copy_pages_past_32_bit_offsets():
    """A pool of more than 2^32 bytes: pages at both ends."""
    P = 2100
    pool = torch.empty(P, 2 * 1024 * 1024, dtype=torch.uint8, device="cuda")
    pool[P - 1] = 7
    pool[5] = 9
    copy_pages([pool], _i32([P - 1, 5]), _i32([0, P - 2]), validate=True)
    assert bool((pool[0] == 7).all()) and bool((pool[P - 2] == 9).all())


def test_copy_pages_leaves_out_clashing_pairs():
    g = _gen(2)
    c = _caches(20, g, ("scale",))[0]
    before = c.clone()
    # 0->1 and 2->1 (second destination), 3->4 with 4->5 (4 is read), 6->6 (itself), 7->8 fine
    src, dst = _i32([0, 2, 3, 4, 6, 7, 9]), _i32([1, 1, 4, 5, 6, 8, -1])
    with pytest.raises(IndexError, match="two places"):
        copy_pages([c], src, dst, validate=True)
    want = before.clone()
    for s, d in ((0, 1), (4, 5), (7, 8)):
        want[d] = before[s]
    assert torch.equal(c, want)


def test_copy_pages_bad_ids_raise_and_skip():
    c = torch.arange(40, device="cuda").reshape(10, 4)
    before = c.clone()
    with pytest.raises(IndexError, match="out of range"):
        copy_pages([c], _i32([10, 1, 2]), _i32([0, 2**31 - 1, 3]), validate=True)
    before[3] = before[2]
    assert torch.equal(c, before)


def test_copy_pages_from_int64_and_another_stream():
    c = torch.arange(4000, device="cuda").reshape(100, 40)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        copy_pages([c], torch.tensor([1, 2], device="cuda"), torch.tensor([50, 60], device="cuda"))
    s.synchronize()
    assert torch.equal(c[50], c[1]) and torch.equal(c[60], c[2])


class Pair:
    """DevicePages beside the plain table; every step is applied to both."""

    def __init__(self, P, bs, S, M, seed=0, kinds=("bf16", "scale")):
        self.dev = DevicePages(P, bs, S, M)
        self.py = Pages([[-1] * M for _ in range(S)], [0] * S, [0] * P, bs)
        self.caches = _caches(P, _gen(seed), kinds)

    def step(self, name, *args):
        getattr(self.py, name)(*args)
        more = {"fork": (self.caches,), "compact": (self.caches,)}.get(name, ())
        want = [c.clone() for c in self.caches]
        for s, d in self.py.moves:
            for w, c in zip(want, self.caches):
                w[d] = c[s]
        self.py.moves = []
        got = getattr(self.dev, name)(*[_i32(a) for a in args], *more, validate=False)
        assert self.dev.read_errors() == self.py.flags, name
        self.py.flags = 0
        self.same(name)
        for w, c in zip(want, self.caches):
            assert torch.equal(w, c), name
        return got

    def same(self, name=""):
        assert self.dev.block_tables.tolist() == self.py.tables, name
        assert self.dev.seq_lens.tolist() == self.py.lens, name
        assert self.dev.ref_counts.tolist() == self.py.refs, name


def test_a_beam_search():
    p = Pair(200, 16, 12, 20)
    p.step("reserve", [0, 1, 2], [35, 16, 1])
    p.step("fork", [0, 0, 1, 2], [3, 4, 5, 6])
    p.step("reserve", [0, 3, 4, 5, 6, 1, 2], [1] * 7)
    p.step("free", [0, 5])
    p.step("fork", [3, 3, -1, 4], [0, 5, 7, 8])
    p.step("reserve", [0, 3, 5, 8], [13, 14, 15, 200])
    p.step("free", [3, 4, 3, -1])
    p.step("compact")
    p.step("fork", [8, 0], [9, 10])
    p.step("compact")
    p.step("free", list(range(12)))
    p.step("compact")
    assert sum(p.py.refs) == 0


@pytest.mark.parametrize("seed", range(12))
def test_random_steps(seed):
    rng = np.random.default_rng(seed)
    bs = int(rng.choice([1, 3, 8, 16, 64]))
    S, P, M = int(rng.integers(1, 40)), int(rng.integers(1, 500)), int(rng.integers(1, 30))
    p = Pair(P, bs, S, M, seed, ("scale", "odd") if seed % 2 else ("layer",))
    for _ in range(25):
        n = int(rng.integers(1, S + 1))
        kind = rng.choice(["reserve", "reserve", "fork", "free", "compact"])
        slots = rng.integers(-1, S + (1 if rng.random() < 0.2 else 0), n).tolist()
        if kind == "reserve":
            p.step("reserve", slots, rng.integers(-1 if rng.random() < 0.1 else 0, 3 * bs + 2, n).tolist())
        elif kind == "fork":
            p.step("fork", rng.integers(-1, S, n).tolist(), slots)
        elif kind == "free":
            p.step("free", slots[: max(1, n // 2)])
        else:
            live = p.step("compact")
            assert int(live) == sum(r > 0 for r in p.py.refs)


@pytest.mark.parametrize("P", [1, 4095, 4096, 4097, 50001])
def test_pools_at_the_edges_of_a_tile(P):
    p = Pair(P, 4, 6, max(4, P // 4 + 1), kinds=("scale",))
    p.step("reserve", [0, 1, 2], [P * 4 // 5, P, 3])
    p.step("free", [0])
    p.step("fork", [1, 2], [3, 4])
    p.step("compact")
    p.step("reserve", [5, 0], [P, P])


def test_more_slots_than_threads_of_a_plan():
    S = 2500
    p = Pair(6000, 2, S, 4, kinds=("scale",))
    p.step("reserve", list(range(1200)), [1 + i % 5 for i in range(1200)])
    p.step("fork", list(range(1200)), list(range(1200, 2400)))
    p.step("reserve", list(range(S)), [1] * S)
    p.step("free", list(range(0, S, 3)))
    p.step("compact")


def test_tables_with_wide_rows_and_an_odd_address():
    base = torch.full((6, 11), -1, dtype=torch.int32, device="cuda")
    refs = torch.zeros(41, dtype=torch.int32, device="cuda")[1:]  # 4 bytes off a 16-byte boundary
    pages = DevicePages.from_tensors(base[:, :7], torch.zeros(6, dtype=torch.int32, device="cuda"), refs, block_size=3)
    py = Pages([[-1] * 7 for _ in range(6)], [0] * 6, [0] * 40, 3)
    for name, args in (("reserve", ([0, 1], [19, 21])), ("fork", ([0, 1], [2, 3])), ("free", ([0],)),
                       ("compact", ())):
        getattr(py, name)(*args)
        getattr(pages, name)(*[_i32(a) for a in args], validate=True)
        assert pages.block_tables.tolist() == py.tables and pages.ref_counts.tolist() == py.refs
    assert bool((base[:, 7:] == -1).all())


def test_exhaustion_leaves_the_slot_and_raises():
    pages = DevicePages(3, 4, 4, 8)
    with pytest.raises(RuntimeError, match="free pages"):
        pages.reserve(_i32([0, 1]), _i32([8, 8]), validate=True)
    assert pages.seq_lens.tolist() == [8, 0, 0, 0]
    assert pages.ref_counts.tolist() == [1, 1, 0]
    pages.reserve(_i32([1]), _i32([3]))
    pages.fork(_i32([1]), _i32([2]))
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="free pages"):
        pages.free(_i32([3]))
    assert pages.seq_lens.tolist() == [8, 3, 0, 0]


def test_a_captured_step_replays():
    """free + fork + reserve in a graph: replays act on the tables as they are then."""
    p = Pair(300, 16, 8, 30)
    p.step("reserve", [0, 1, 2, 3], [40, 17, 64, 5])
    parents, children, one = _i32([0, 1, 2, 3]), _i32([4, 5, 6, 7]), _i32([1] * 8)
    slots = _i32(list(range(8)))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        p.dev.free(children)
        p.dev.fork(parents, children, p.caches)
        p.dev.reserve(slots, one)
    for _ in range(20):
        p.py.free([4, 5, 6, 7])
        p.py.fork([0, 1, 2, 3], [4, 5, 6, 7])
        p.py.reserve(list(range(8)), [1] * 8)
        graph.replay()
        p.same()
    assert p.dev.read_errors() == 0


def test_refusals():
    with pytest.raises(ValueError):
        DevicePages(0, 16, 4, 4)
    with pytest.raises(RuntimeError):
        DevicePages(4, 16, 4, 4, "cpu")
    pages = DevicePages(8, 16, 4, 4)
    with pytest.raises(ValueError, match="at most 4"):
        pages.free(_i32([0, 1, 2, 3, 0]))
    with pytest.raises(ValueError, match="children"):
        pages.fork(_i32([0]), _i32([1, 2]))
    with pytest.raises(ValueError, match="8 blocks"):
        pages.fork(_i32([0]), _i32([1]), [torch.zeros(9, 4, device="cuda")])
    with pytest.raises(ValueError, match="at most"):
        copy_pages([torch.zeros(4, 4, device="cuda")] * 9, _i32([0]), _i32([1]))
    with pytest.raises(ValueError, match="one strided"):
        copy_pages([torch.zeros(4, 8, 8, 8, device="cuda")[:, ::2, ::2]], _i32([0]), _i32([1]))
    with pytest.raises(ValueError, match="overlap"):
        copy_pages([torch.zeros(1, 4, device="cuda").expand(4, 4)], _i32([0]), _i32([1]))
    with pytest.raises(ValueError):
        copy_pages([], _i32([0]), _i32([1]))
    with pytest.raises(ValueError):
        copy_pages([torch.zeros(4, 4)], _i32([0]), _i32([1]))
    copy_pages([torch.zeros(4, 4, device="cuda")], _i32([]), _i32([]))
