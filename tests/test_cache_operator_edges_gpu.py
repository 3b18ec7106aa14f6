"""Edges of the operators over a paged cache: padding pairs among forks, block ids outside
the pool, empty slots, error words read while other streams report, workspaces,
values that are not finite, rows without keys, blocks of zeros."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from _ops64 import F8, Pages, attend64, check
from llm_serving_runtime_b200 import (
    DevicePages,
    PrefixGroups,
    ScoreModifiers,
    _lib,
    copy_pages,
    kv_append,
    paged_attention,
    paged_attention_decode,
    read_device_errors,
)
from llm_serving_runtime_b200.kv_block_pool import Fp8KVBlockPool, write_tokens_batch_into

pytestmark = pytest.mark.gpu
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _pages_beside_the_plain_table(P, bs, S, M):
    return DevicePages(P, bs, S, M), Pages([[-1] * M for _ in range(S)], [0] * S, [0] * P, bs)


def _step(pages, table, name, *args):
    getattr(table, name)(*args)
    table.moves = []
    getattr(pages, name)(*[_i32(a) for a in args], validate=False)
    assert pages.read_errors() == table.flags
    table.flags = 0
    assert pages.block_tables.tolist() == table.tables
    assert pages.seq_lens.tolist() == table.lens and pages.ref_counts.tolist() == table.refs


def test_a_padding_pair_does_not_claim_its_child():
    """A pair without a parent is padding whatever its child is: a later pair may name it."""
    pages, table = _pages_beside_the_plain_table(20, 4, 6, 5)
    _step(pages, table, "reserve", [0, 1], [6, 9])
    _step(pages, table, "fork", [-1, 0, -1], [3, 3, 3])
    assert table.lens[3] == 6
    _step(pages, table, "fork", [-1, -1, 1, 1, 0], [4, 5, 5, 5, 4])  # 5 a second time is an error
    assert table.lens[4:] == [6, 9]


@pytest.mark.parametrize("seed", range(8))
def test_forks_among_padding_pairs(seed):
    rng = np.random.default_rng(seed)
    S = int(rng.integers(4, 1500))
    pages, table = _pages_beside_the_plain_table(4 * S, 3, S, 3)
    full = S // 3
    _step(pages, table, "reserve", list(range(full)), rng.integers(1, 7, full).tolist())
    for _ in range(4):
        n = int(rng.integers(2, S + 1))
        parents = np.where(rng.random(n) < 0.5, -1, rng.integers(0, full, n))
        children = rng.integers(full, S, n)
        _step(pages, table, "fork", parents.tolist(), children.tolist())
        _step(pages, table, "free", rng.permutation(np.arange(full, S))[: (S - full) // 2].tolist())


def _attend_case(cache, lens, q, Hq, Hkv, D, bs, seed):
    """(query, kc, vc, tables, lens, scale keywords); the pool's last block holds zeros
    (of scale 0), and no table names it."""
    g = torch.Generator().manual_seed(seed)
    n = [(x + q + bs - 1) // bs for x in lens]
    nb = sum(n) + 1
    tables = torch.zeros(len(lens), max(n), dtype=torch.int32)
    at = 0
    for b, k in enumerate(n):
        tables[b, :k] = torch.arange(at, at + k)
        at += k
    dt = BF if cache == F8 else cache
    query = torch.randn(len(lens), Hq, q, D, generator=g).to(dt).cuda()
    kc, vc = ((torch.randn(nb, Hkv, bs, D, generator=g) * 4).to(cache) for _ in range(2))
    kc.view(torch.uint8)[-1] = vc.view(torch.uint8)[-1] = 0
    kw = {}
    if cache == F8:
        for name in ("key_scales", "value_scales"):
            s = torch.rand(nb, Hkv, generator=g) + 0.25
            s[-1] = 0
            kw[name] = s.cuda()
    return query, kc.cuda(), vc.cuda(), tables, _i32(lens), kw


@pytest.mark.parametrize("q,B", [(1, 6), (1, 20), (3, 40), (40, 20), (40, 40)])
@pytest.mark.parametrize("cache,D", [(FP, 32), (FP, 33), (FP, 64), (FP, 128), (BF, 64), (HF, 128), (F8, 64)])
def test_a_bad_block_counts_as_zeros(cache, D, q, B):
    """A block id outside the pool is flagged and read as zeros, never as what the shared
    memory of the GPU still holds: the same bits as a block of zeros, call after call."""
    lens = [70, 16, 5, 300] + [90 + 7 * i for i in range(B - 4)]
    query, kc, vc, tables, lens, kw = _attend_case(cache, lens, q, 8, 4, D, 16, 31)
    nb = kc.shape[0]
    where = [(0, 0), (0, 2), (1, 0), (3, 1), (3, 7), (3, 18), (5, 3)]
    zeros = tables.clone()
    for b, i in where:
        zeros[b, i] = nb - 1
    mods = ScoreModifiers(softcap=20.0)
    want = paged_attention_decode(query, kc, vc, zeros.cuda(), lens, 0.2, score_modifiers=mods, validate=True, **kw)
    assert bool(want.isfinite().all())
    for bad in (-1, nb, nb + 1000):
        wrong = tables.clone()
        for b, i in where:
            wrong[b, i] = bad
        wrong = wrong.cuda()
        for _ in range(3):
            # fills shared memory with other numbers
            paged_attention_decode(query, kc * 3 if cache != F8 else kc, vc, tables.cuda(), lens, 0.2,
                                   score_modifiers=mods, **kw)
            out = paged_attention_decode(query, kc, vc, wrong, lens, 0.2, score_modifiers=mods, validate=False, **kw)
            assert read_device_errors() & 0x1
            assert torch.equal(out, want)


@pytest.mark.parametrize("q", [1, 3])
@pytest.mark.parametrize("cache", [BF, HF, FP, F8])
def test_a_loop_over_slots_some_of_which_are_empty(cache, q):
    """The whole table of a DevicePages goes into the call: a slot of length 0 has no new
    tokens, its rows are zero, nothing is written for it and nothing reported."""
    g = torch.Generator().manual_seed(5)
    P, bs, S, M, Hq, Hkv, D = 40, 16, 6, 8, 8, 2, 64
    dt = BF if cache == F8 else cache
    pages = DevicePages(P, bs, S, M)
    live = [1, 4]
    pages.reserve(_i32(live), _i32([40, 15]), validate=True)
    kw = {"score_modifiers": ScoreModifiers(softcap=30.0)}
    if cache == F8:
        pool = Fp8KVBlockPool(P, 1, Hkv, bs, D)
        kc, vc = pool.k_layer_view(0), pool.v_layer_view(0)
        kw.update(key_scales=pool.k_layer_scales(0), value_scales=pool.v_layer_scales(0))
    else:
        kc, vc = (torch.randn(P, Hkv, bs, D, generator=g).to(cache).cuda() for _ in range(2))
    forms = [kw] if cache == F8 else [kw, {}]  # plain attention too
    for step in range(4):
        if step == 2:
            pages.free(_i32([4]), validate=True)
            live = [1]
        pages.reserve(_i32(live), _i32([q] * len(live)), validate=True)
        query = torch.randn(S, Hq, q, D, generator=g).to(dt).cuda()
        key, value = (torch.randn(S, Hkv, q, D, generator=g).to(dt).cuda() for _ in range(2))
        rows = torch.tensor(live).cuda()
        for form in forms:
            state = [t.clone() for t in (kc, vc, *(form[s] for s in ("key_scales", "value_scales") if s in form))]
            outs, caches = [], []
            for validate in (True, None):
                for t, s in zip((kc, vc, form.get("key_scales"), form.get("value_scales")), state):
                    t.copy_(s)
                outs.append(paged_attention_decode(query, kc, vc, pages.block_tables, pages.seq_lens, 0.125, key=key,
                                                   value=value, context_lens_include_new=True, validate=validate,
                                                   **form))
                caches.append([t.float() for t in (kc, vc)])
            assert read_device_errors() == 0
            for t, s in zip((kc, vc, form.get("key_scales"), form.get("value_scales")), state):
                t.copy_(s)
            want = paged_attention_decode(query[rows], kc, vc, pages.block_tables[rows], pages.seq_lens[rows], 0.125,
                                          key=key[rows], value=value[rows], context_lens_include_new=True,
                                          validate=True, **form)
            for out, cache_after in zip(outs, caches):
                # plain 16-bit attention splits its work by the batch: both sides round their
                # weights (2^-11 at most) and their outputs
                bar = 0.0 if form or cache == FP else float(torch.finfo(dt).eps * want.abs().max()
                                                            + 2.0**-10 * max(vc.abs().max(), value.abs().max()))
                assert float((out[rows] - want).abs().max()) <= bar
                assert sum(int(x) for x in out.abs().sum((1, 2, 3)) != 0) == len(live)
                for a, t in zip(cache_after, (kc, vc)):
                    assert torch.equal(a, t.float())


@pytest.mark.parametrize("cache", [BF, F8])
def test_other_tokens_before_the_start_are_still_reported(cache):
    """Only a whole row of length 0 is empty: a negative position, or a length that is less
    than its new tokens, stays an error."""
    P, bs, Hkv, D = 6, 16, 2, 64
    kc, vc = (torch.zeros(P, Hkv, bs, D, device="cuda").to(cache) for _ in range(2))
    kw = {n: torch.zeros(P, Hkv, device="cuda") for n in ("key_scales", "value_scales")} if cache == F8 else {}
    rows = torch.ones(2, Hkv, 2, D, dtype=BF, device="cuda")
    tables = _i32([[1, 2], [3, 4]])

    def append(positions, offset):
        kv_append(rows, rows, kc, vc, block_tables=tables, positions=_i32(positions), position_offset=offset,
                  validate=True, **kw)

    append([0, 5], -2)  # length 0, and a row whose two tokens are its last
    for positions, offset in (([1, 5], -2), ([0, 5], -1), ([-2, 5], 0), ([-1, 5], -2)):
        with pytest.raises(IndexError, match="slot"):
            append(positions, offset)


class _OtherStream:
    """An error word seen by a host whose every look is followed at once by a report of a
    kernel on another stream (here a new bit is set in the same memory)."""

    def __init__(self, word):
        self.word, self.reported, self.bits = word, 0, [0x100, 0x40, 0x20, 0x10]

    @property
    def value(self):
        seen = self.word.value
        self.reported |= self.bits[0]
        self.word.value = seen | self.bits.pop(0)
        return seen

    @value.setter
    def value(self, new):
        self.word.value = new


def test_no_report_is_lost_between_a_look_and_the_clearing(monkeypatch):
    pages = DevicePages(8, 4, 4, 4)
    word = pages._word
    real = word.word
    pages.reserve(_i32([9]), _i32([1]), validate=False)  # a slot outside the table: 0x80
    torch.cuda.synchronize()
    assert real.value == 0x80
    other = _OtherStream(real)
    monkeypatch.setattr(word, "word", other)
    seen = word.take() if word.word.value else 0  # as the next call looks and then clears
    monkeypatch.setattr(word, "word", real)
    assert seen | word.take() == 0x80 | other.reported
    assert word.take() == 0 and pages.read_errors() == 0


def test_reading_the_devices_errors_loses_no_report(monkeypatch):
    c = torch.zeros(8, 4, device="cuda")
    copy_pages([c], _i32([1]), _i32([2]), validate=True)
    word = paged_attention._host_words[0]
    assert read_device_errors() == 0
    real = word.word
    copy_pages([c], _i32([99]), _i32([2]), validate=False)
    torch.cuda.synchronize()
    other = _OtherStream(real)
    monkeypatch.setattr(word, "word", other)
    seen = read_device_errors()
    monkeypatch.setattr(word, "word", real)
    assert seen & 0x1
    assert seen | read_device_errors() == 0x1 | other.reported
    assert word.take() == 0


def test_an_error_that_another_thread_took_does_not_raise_again(monkeypatch):
    c = torch.zeros(8, 4, device="cuda")
    copy_pages([c], _i32([1]), _i32([2]), validate=True)
    word = paged_attention._host_words[0]
    real = word.word

    class Taken:  # the look sees a bit, and another thread takes it before this one can
        @property
        def value(self):
            return 0x1

        @value.setter
        def value(self, new):
            real.value = new

    monkeypatch.setattr(word, "word", Taken())
    try:
        word.raise_landed()
    finally:
        monkeypatch.setattr(word, "word", real)


def test_errors_reported_while_others_are_read():
    """Two streams report, one after each reading of the other's: every report raises
    somewhere, and none twice."""
    c = torch.zeros(8, 4, device="cuda")
    copy_pages([c], _i32([1]), _i32([2]), validate=True)
    word = paged_attention._host_words[0]
    bad = [(_i32([99]), _i32([2])), (_i32([1, 1]), _i32([3, 3]))]
    streams = [torch.cuda.Stream() for _ in bad]
    torch.cuda.synchronize()
    for _ in range(50):
        seen = 0
        for s, (src, dst) in zip(streams, bad):
            with torch.cuda.stream(s):
                copy_pages([c], src, dst, validate=False)
                seen |= word.take()
        torch.cuda.synchronize()
        seen |= word.take()
        assert seen == 0x41
    assert word.take() == 0


@pytest.fixture
def fresh_workspaces(monkeypatch):
    """No workspace yet, as in a new process."""
    for name, value in (("_workspaces", {}), ("_outgrown", []), ("_captured", set())):
        monkeypatch.setattr(paged_attention, name, value)
    yield paged_attention._workspaces
    torch.cuda.synchronize()


def _fp32_case(B=3):
    g = torch.Generator().manual_seed(6)
    kc, vc = (torch.randn(20, 2, 16, 64, generator=g).cuda() for _ in range(2))
    query = torch.randn(B, 4, 1, 64, generator=g).cuda()
    return query, kc, vc, torch.randint(0, 20, (B, 4), generator=g).int().cuda(), _i32([50, 3, 17][:B]), 0.125


def test_plain_fp32_decode_asks_for_no_more_than_its_header(fresh_workspaces):
    need = _lib.load().pa_decode_workspace_bytes(3, 4, 2, 1, 64, _lib.PA_DTYPE_FLOAT32, 0)
    assert need == 256
    args = _fp32_case()
    paged_attention.decode_workspace(torch.device("cuda", 0))  # what any earlier call leaves
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):  # no eager call of this kind before
        out = paged_attention_decode(*args)
    graph.replay()
    torch.cuda.synchronize()
    ws = fresh_workspaces[0]
    assert ws.numel() == 256
    got = out.clone()
    assert torch.equal(got, paged_attention_decode(*args, validate=True))
    assert fresh_workspaces[0] is ws
    # changed scores bring their own need
    capped = paged_attention_decode(*args, score_modifiers=ScoreModifiers(softcap=1e4), validate=True)
    assert fresh_workspaces[0].numel() > 256
    assert float((capped - got).abs().max()) < 1e-3
    for _ in range(2):  # the short way finds a workspace that fits
        assert torch.equal(capped, paged_attention_decode(*args, score_modifiers=ScoreModifiers(softcap=1e4)))


def test_a_workspace_of_the_plain_size_is_refused_for_changed_fp32_scores():
    args = _fp32_case()
    with pytest.raises(RuntimeError, match="workspace too small"):
        paged_attention_decode(*args, score_modifiers=ScoreModifiers(window=3),
                               workspace=torch.zeros(256, dtype=torch.uint8, device="cuda"))


def test_an_outgrown_workspace_is_kept_for_captured_graphs_alone(fresh_workspaces):
    dev = torch.device("cuda", 0)
    first = paged_attention.decode_workspace(dev, 1000)
    second = paged_attention.decode_workspace(dev, 5000)
    third = paged_attention.decode_workspace(dev, 6000)
    assert (first.numel(), second.numel(), third.numel()) == (1000, 5000, 6000)
    assert not paged_attention._outgrown
    assert paged_attention.decode_workspace(dev, 100) is third
    graph, args = torch.cuda.CUDAGraph(), _fp32_case()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = paged_attention_decode(*args)
    fourth = paged_attention.decode_workspace(dev, 7000)
    assert [w.data_ptr() for w in paged_attention._outgrown] == [third.data_ptr()]
    assert fourth.numel() >= 12000  # what is kept stays below what is used
    fifth = paged_attention.decode_workspace(dev, fourth.numel() + 1)
    assert len(paged_attention._outgrown) == 1 and fifth.numel() == fourth.numel() + 1
    graph.replay()
    assert torch.equal(out, paged_attention_decode(*args, validate=True))


@pytest.mark.parametrize("short", [True, False])
def test_a_graph_of_an_extended_call_keeps_its_workspace(fresh_workspaces, monkeypatch, short):
    """Captured in one extension call or through the checks: growing the workspace later
    takes nothing from the graph."""
    if not short:
        monkeypatch.setattr(paged_attention, "_VALIDATE_DEFAULT", True)
    args, mods = _fp32_case(), ScoreModifiers(softcap=3.0)
    for _ in range(2):
        want = paged_attention_decode(*args, score_modifiers=mods)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged_attention_decode(*args, score_modifiers=mods)
    ws = fresh_workspaces[0]
    paged_attention.decode_workspace(ws.device, 3 * ws.numel())
    assert [w.data_ptr() for w in paged_attention._outgrown] == [ws.data_ptr()]
    graph.replay()
    assert torch.equal(out, want)


def _chunk_case(dtype, B, q, L, Hkv, G, D, bs, seed):
    g = torch.Generator().manual_seed(seed)
    n = (L + q + bs - 1) // bs
    nb = B * n
    tables = torch.randperm(nb, generator=g).int().reshape(B, n)
    kc, vc = (torch.randn(nb, Hkv, bs, D, generator=g).to(dtype).cuda() for _ in range(2))
    query = torch.randn(B, Hkv * G, q, D, generator=g).to(dtype).cuda()
    return query, kc, vc, tables, torch.full((B,), L, dtype=torch.int32)


def _put(cache, tables, bs, b, pos, col, value):
    cache[int(tables[b, pos // bs]), :, pos % bs, col] = value


@pytest.mark.parametrize("dtype,D,bs", [(BF, 64, 16), (BF, 128, 8), (HF, 128, 64), (HF, 72, 16)])
@pytest.mark.parametrize("kind", ["causal", "window", "documents", "prefix"])
def test_values_that_are_not_finite_reach_the_rows_that_see_them(dtype, D, bs, kind):
    """Prefill chunks on the tcgen05 kernel: infinities and NaN among values that some of a
    tile's rows see and others do not, from one of them to every key of a sequence.  They
    stand in one column each, so the others show that nothing else changes."""
    B, q, L, Hkv, G = 19, 40, 100, 8, 2
    query, kc, vc, tables, lens = _chunk_case(dtype, B, q, L, Hkv, G, D, bs, 41)
    rng = np.random.default_rng(3)
    some = [float("inf"), -float("inf"), float("nan")]
    new = np.arange(L, L + q)
    seen_in_part = {"causal": new, "window": np.concatenate([np.arange(L - 50, L - 10), new]),
                    "documents": np.arange(L + q), "prefix": np.arange(L + 8, L + q)}[kind]
    for b in range(B):
        n = [0, 1, 2, 7, 40][b % 5]
        if b == 4:
            where = seen_in_part
        else:
            where = rng.permutation(seen_in_part)[:n]
        for pos in where:
            _put(vc, tables, bs, b, int(pos), int(rng.integers(0, D)), some[int(rng.integers(0, 3))])
    for pos in (L + 3, L + 20):  # a key of its own that is not finite: its rows are NaN
        _put(kc, tables, bs, 7, pos, 1, float("nan"))
        _put(vc, tables, bs, 7, pos, 2, float("inf"))
    args = {"softcap": 20.0}
    if kind == "window":
        args["window"] = 50
    elif kind == "documents":
        pos = torch.arange(L, L + q)[None].repeat(B, 1)
        args["key_starts"] = (pos // 9 * 9 - (pos % 9 == 0) * 60).clamp_min(0).int().cuda()
    elif kind == "prefix":
        args["prefix_lens"] = torch.full((B,), L + 8, dtype=torch.int32, device="cuda")
    mods = ScoreModifiers(alibi_slopes=torch.linspace(0, 0.2, Hkv * G).cuda(), **args)
    out = paged_attention_decode(query, kc, vc, tables.cuda(), lens.cuda(), 0.1, score_modifiers=mods, validate=True)
    assert _lib.last_kernel() == "pa::prefill_umma_kernel<scored>"
    ref, bar = attend64(query, kc, vc, tables, lens, 0.1, alibi_slopes=mods.alibi_slopes, **args)
    assert bool(torch.isnan(ref).any()) and bool(torch.isinf(ref).any())
    o = out.double().cpu()
    assert torch.equal(torch.isinf(o) * o.sign().nan_to_num(), torch.isinf(ref) * ref.sign().nan_to_num())
    assert torch.equal(torch.isnan(o), torch.isnan(ref))
    fine = torch.isfinite(ref)
    check(o.where(fine, 0.0), ref.where(fine, 0.0), bar.where(fine, 0.0))
    for _ in range(3):
        again = paged_attention_decode(query, kc, vc, tables.cuda(), lens.cuda(), 0.1, score_modifiers=mods)
        assert torch.equal(out.view(torch.int16), again.view(torch.int16))


def test_one_value_that_is_not_finite_costs_little():
    """A call over long cached contexts takes about as long with an infinite value among
    its new tokens as without (a hundred times as long when the rows of its tile are
    worked out anew)."""
    B, q, L, bs = 8, 256, 8192, 16
    n = (L + q + bs - 1) // bs
    g = torch.Generator(device="cuda").manual_seed(5)
    kc, vc = (torch.randn(B * n, 8, bs, 128, generator=g, device="cuda").to(BF) for _ in range(2))
    query = torch.randn(B, 32, q, 128, generator=g, device="cuda").to(BF)
    tables = torch.arange(B * n, dtype=torch.int32, device="cuda").reshape(B, n)
    lens, mods = _i32([L] * B), ScoreModifiers(softcap=50.0)

    def best():
        took = []
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            paged_attention_decode(query, kc, vc, tables, lens, 0.09, score_modifiers=mods)
            b.record()
            b.synchronize()
            took.append(a.elapsed_time(b))
        return min(took)

    clean = best()
    vc[int(tables[0, (L + 100) // bs]), :, (L + 100) % bs, 3] = float("inf")
    assert best() < 5 * clean


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 72, 128])
@pytest.mark.parametrize("scored", [True, False])
def test_rows_without_keys_are_zero_on_the_multi_query_kernel(scored, D, dtype):
    """Sequences of length 0 and tokens before a sequence's start, whole tiles of them: zeros,
    not what a tile's queries left where its rows are stored from."""
    B, q, Hkv, G, bs = 40, 64, 4, 8, 16
    g = torch.Generator().manual_seed(43)
    nb = 200
    kc, vc = (torch.randn(nb, Hkv, bs, D, generator=g).to(dtype).cuda() for _ in range(2))
    tables = torch.randint(0, nb, (B, 8), generator=g).int().cuda()
    query = torch.randn(B, Hkv * G, q, D, generator=g).to(dtype).cuda()
    lens = torch.tensor([[0, 20, -3, 64, 100, 1, 33, 0][b % 8] for b in range(B)])
    kw = {"score_modifiers": ScoreModifiers(softcap=30.0)} if scored else {}
    want = None
    for _ in range(20):
        out = paged_attention_decode(query, kc, vc, tables, _i32(lens.tolist()), 0.1, context_lens_include_new=True,
                                     validate=True, **kw)
        assert _lib.last_kernel() == "pa::prefill_umma_kernel" + ("<scored>" if scored else "")
        for b, n in enumerate(lens.tolist()):
            empty = q - min(max(n, 0), q)  # tokens before the start
            assert not bool(out[b, :, :empty].any()), b
            assert n <= 0 or bool((out[b, :, empty:] != 0).any())
        want = out if want is None else want
        assert torch.equal(out, want)


@pytest.mark.parametrize("B,q,L,M,kernel", [(2, 1, 300, 20, "pa::decode_direct_kernel<few>"),
                                            (1, 5, 5000, 400, "pa::decode_direct_kernel<few>"),
                                            (40, 1, 300, 20, "pa::decode_direct_kernel<many>"),
                                            (40, 1, 300, 300, "pa::decode_mma_kernel<ext>"),
                                            (20, 40, 200, 20, "pa::prefill_mma_kernel<ext>")])
@pytest.mark.parametrize("scored", [True, False])
def test_blocks_of_zeros_beside_huge_values(scored, B, q, L, M, kernel):
    """A block of zeros (a scale of 0, or the append's least, 2^-100) has its weight in the
    norm beside blocks of any scale up to 2^60, in whichever order they come."""
    Hkv, G, D, bs = 8, 2, 64, 16
    g = torch.Generator().manual_seed(44)
    per = (L + q + bs - 1) // bs
    nb = B * per
    tables = torch.zeros(B, M, dtype=torch.int32)
    tables[:, :per] = torch.arange(nb).reshape(B, per)
    kc, vc = ((torch.randn(nb, Hkv, bs, D, generator=g) * 100).clamp(-448, 448).to(F8) for _ in range(2))
    ks = torch.exp2(torch.randint(-9, -6, (nb, Hkv), generator=g).float())
    vs = torch.exp2(torch.randint(-9, -6, (nb, Hkv), generator=g).float())
    kind = torch.randint(0, 6, (nb, Hkv), generator=g)
    vs[kind == 1] = 0
    vs[kind == 2] = 2.0**-100
    vs[kind == 3] = 2.0 ** float([32, 45, 60][B % 3])
    vs[:per:2] = 0  # a row of whole zeros up to its end
    vs[per - 1] = 2.0**33
    kind[1::7] = 2  # its codes are 0 as well
    vs[1::7] = 2.0**-100
    vc.view(torch.uint8)[1::7] = 0
    query = torch.randn(B, Hkv * G, q, D, generator=g).to(BF).cuda()
    lens = torch.full((B,), L, dtype=torch.int32)
    state = [t.cuda() for t in (kc, vc)]
    kw = {"key_scales": ks.cuda(), "value_scales": vs.cuda()}
    mods = {"softcap": 20.0} if scored else {}
    out = paged_attention_decode(query, *state, tables.cuda(), lens.cuda(), 0.05, validate=True,
                                 score_modifiers=ScoreModifiers(**mods) if scored else None, **kw)
    assert _lib.last_kernel() == kernel
    ref, bar = attend64(query, *state, tables, lens, 0.05, **kw, **mods)
    check(out, ref, bar)


def test_a_batched_write_takes_each_view_of_the_pool_once():
    class Counting:
        def __init__(self, pool):
            self.pool, self.taken = pool, []

        def __getattr__(self, name):
            if name.startswith(("k_layer", "v_layer")):
                self.taken.append(name)
            return getattr(self.pool, name)

    pool = Counting(Fp8KVBlockPool(4, 2, 2, 16, 64))
    rows = torch.ones(1, 2, 3, 64, dtype=BF, device="cuda")
    write_tokens_batch_into(pool, 1, torch.tensor([[2, 3]]), torch.tensor([15]), rows, rows)
    assert sorted(pool.taken) == ["k_layer_scales", "k_layer_view", "v_layer_scales", "v_layer_view"]
    torch.cuda.synchronize()
    got = pool.pool.k.float() * pool.pool.k_scales[..., None, None]
    assert got[2, 1, :, 15].eq(1).all() and got[3, 1, :, :2].eq(1).all() and int(got.count_nonzero()) == 2 * 3 * 64


@pytest.mark.parametrize("D", [64, 128])
def test_empty_parts_of_a_prefix_take_nothing_from_the_queries(D):
    """A short shared prefix beside a long one, whose splits it leaves empty: an infinite query
    of one member does not reach the others of its tile."""
    Hkv, G, bs, q = 8, 4, 16, 1
    g = torch.Generator().manual_seed(45)
    prefixes, sizes = [64, 4096], [5, 2]
    rows = [list(range(5)), [5, 6]]
    lens = [70, 64, 90, 75, 200, 4100, 4096]
    M = (max(lens) + q + bs - 1) // bs
    tables, at = torch.zeros(7, M, dtype=torch.int32), 0
    for prefix, members in zip(prefixes, rows):
        shared = torch.arange(at, at + prefix // bs)
        at += prefix // bs
        for r in members:
            tables[r, : prefix // bs] = shared
            n = (lens[r] + q + bs - 1) // bs - prefix // bs
            tables[r, prefix // bs: prefix // bs + n] = torch.arange(at, at + n)
            at += n
    kc, vc = (torch.randn(at, Hkv, bs, D, generator=g).to(BF).cuda() for _ in range(2))
    query = torch.randn(sum(sizes), Hkv * G, q, D, generator=g).to(BF).cuda()
    groups = PrefixGroups.from_members(rows, prefixes, 7, "cuda")
    args = (kc, vc, tables.cuda(), _i32(lens), D**-0.5)
    want = paged_attention_decode(query, *args, prefix_groups=groups, validate=True)
    assert bool(want.isfinite().all())
    query[2] = float("inf")
    others = torch.tensor([0, 1, 3, 4, 5, 6]).cuda()
    for _ in range(20):
        out = paged_attention_decode(query, *args, prefix_groups=groups, validate=True)
        assert torch.equal(out[others], want[others])
