"""The operators over a paged cache together, as a decode loop uses them: pages reserved,
forked, freed and compacted on the device, rows appended in 8 bits, attended with
changed scores; in one extension call, through the checks, and in a captured graph."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from _ops64 import F8, Pages, append8, attend64, check
from llm_serving_runtime_b200 import (
    DevicePages,
    ScoreModifiers,
    _lib,
    copy_pages,
    kv_append,
    paged_attention,
    paged_attention_decode,
    read_device_errors,
)
from llm_serving_runtime_b200.kv_block_pool import Fp8KVBlockPool
from llm_serving_runtime_b200.shared_blocks import BlockRefAllocator

pytestmark = pytest.mark.gpu
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _bits(t):
    return t.view(torch.uint8) if t.dtype == F8 else t


def _random_pool(g, nb, layers, H, bs, D):
    pool = Fp8KVBlockPool(nb, layers, H, bs, D)
    for c in (pool.k, pool.v):
        c.copy_((torch.randn(c.shape, generator=g) * 100).clamp(-448, 448).to(F8))
    for s in (pool.k_scales, pool.v_scales):
        s.copy_(torch.exp2(torch.randint(-9, -5, s.shape, generator=g).float()))
    return pool


class Loop:
    """A beam search of four sequences over an 8-bit pool, a step at a time: the lower
    half of the beams is replaced by forks of the upper half, all grow by a token."""

    P, bs, S, layers, Hq, Hkv, D = 90, 16, 4, 2, 8, 2, 64

    def __init__(self, seed):
        g = torch.Generator().manual_seed(seed)
        self.pool = _random_pool(g, self.P, self.layers, self.Hkv, self.bs, self.D)
        self.pages = DevicePages(self.P, self.bs, self.S, 12)
        self.pages.reserve(_i32([0, 1, 2, 3]), _i32([40, 31, 17, 80]))
        self.mods = ScoreModifiers(softcap=15.0, window=48, alibi_slopes=torch.rand(self.Hq, generator=g).cuda() / 8)
        shape = (self.layers, self.S)
        self.q = torch.empty(*shape, self.Hq, 1, self.D, dtype=BF, device="cuda")
        self.k, self.v = (torch.empty(*shape, self.Hkv, 1, self.D, dtype=BF, device="cuda") for _ in range(2))
        self.out = torch.empty_like(self.q)
        self.parents, self.children = _i32([0, 1]), _i32([2, 3])
        self.all, self.one = _i32([0, 1, 2, 3]), _i32([1] * 4)

    def new_rows(self, g):
        for t in (self.q, self.k, self.v):
            t.copy_(torch.randn(t.shape, generator=g))

    def step(self, **kw):
        self.pages.free(self.children, **kw)
        self.pages.fork(self.parents, self.children, self.pool.caches, **kw)
        self.pages.reserve(self.all, self.one, **kw)
        for i in range(self.layers):
            paged_attention_decode(
                self.q[i], self.pool.k_layer_view(i), self.pool.v_layer_view(i), self.pages.block_tables,
                self.pages.seq_lens, self.D**-0.5, key=self.k[i], value=self.v[i], out=self.out[i],
                context_lens_include_new=True, key_scales=self.pool.k_layer_scales(i),
                value_scales=self.pool.v_layer_scales(i), score_modifiers=self.mods, **kw)

    def state(self):
        return [self.out, self.pages.block_tables, self.pages.seq_lens, self.pages.ref_counts] + \
            [_bits(c) for c in self.pool.caches]


def test_a_beam_search_over_an_8_bit_cache():
    """Checked, unchecked and replayed runs agree bit for bit, the tables with the plain
    ones, the cache with the plain append, the outputs with 64 bits."""
    runs = {kind: Loop(1) for kind in ("checked", "plain", "graph")}
    first = runs["checked"]
    table = Pages(first.pages.block_tables.tolist(), first.pages.seq_lens.tolist(), first.pages.ref_counts.tolist(),
                  Loop.bs)
    mirror = [c.double().cpu().numpy() if c.dtype == F8 else c.cpu().numpy() for c in first.pool.caches]
    gens = {kind: torch.Generator().manual_seed(2) for kind in runs}
    graph = None
    for step in range(40):
        for kind, run in runs.items():
            run.new_rows(gens[kind])
            if kind == "checked":
                run.step(validate=True)
            elif kind == "plain" or step == 0:
                run.step()
            else:
                if graph is None:
                    torch.cuda.synchronize()
                    graph = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(graph):
                        run.step()
                graph.replay()
        # the plain forms
        table.free([2, 3])
        table.fork([0, 1], [2, 3])
        for s, d in table.moves:
            for c in mirror:
                c[d] = c[s]
        table.moves = []
        table.reserve([0, 1, 2, 3], [1] * 4)
        assert table.flags == 0
        bt = torch.tensor(table.tables, dtype=torch.int32)
        lens = torch.tensor(table.lens) - 1
        slots = [table.tables[b][n // Loop.bs] * Loop.bs + n % Loop.bs for b, n in enumerate(lens.tolist())]
        for i in range(Loop.layers):
            for rows, codes, scales in ((first.k, mirror[0], mirror[2]), (first.v, mirror[1], mirror[3])):
                c, s = codes[:, i].copy(), scales[:, i].copy()
                assert append8(rows[i].float().cpu().numpy(), c, s, slots, 1, Loop.bs) == 0
                codes[:, i], scales[:, i] = c, s
        for got, want in zip(first.pool.caches, mirror):
            assert np.array_equal(got.double().cpu().numpy(), want), step
        assert first.pages.block_tables.tolist() == table.tables and first.pages.seq_lens.tolist() == table.lens
        for kind in ("plain", "graph"):
            for a, b in zip(first.state(), runs[kind].state()):
                assert torch.equal(a, b), (step, kind)
        if step % 13 == 0:
            for i in range(Loop.layers):
                ref, bar = attend64(first.q[i], first.pool.k_layer_view(i), first.pool.v_layer_view(i), bt.clamp(min=0),
                                    lens.int(), Loop.D**-0.5, key_scales=first.pool.k_layer_scales(i),
                                    value_scales=first.pool.v_layer_scales(i), softcap=15.0, window=48,
                                    alibi_slopes=first.mods.alibi_slopes)
                check(first.out[i], ref, bar)
    # a compaction between steps: the same sequences under other page ids
    before = first.out.clone()
    live = first.pages.compact(first.pool.caches, validate=True)
    assert table.compact() == int(live) and first.pages.block_tables.tolist() == table.tables
    for i in range(Loop.layers):
        paged_attention_decode(
            first.q[i], first.pool.k_layer_view(i), first.pool.v_layer_view(i), first.pages.block_tables,
            first.pages.seq_lens, Loop.D**-0.5, out=first.out[i], context_lens_include_new=True,
            key_scales=first.pool.k_layer_scales(i), value_scales=first.pool.v_layer_scales(i),
            score_modifiers=first.mods, validate=True)
    assert torch.equal(before, first.out)
    assert read_device_errors() == 0 and all(r.pages.read_errors() == 0 for r in runs.values())


class Spy:
    """Stands in front of the extension and notes what each call answered."""

    def __init__(self):
        self.host, self.answers = _lib.host(), []

    def __getattr__(self, name):
        def call(*args):
            got = getattr(self.host, name)(*args)
            self.answers.append((name, got is not None))
            return got
        return call


@pytest.fixture
def spy(monkeypatch):
    from llm_serving_runtime_b200 import device_pages

    s = Spy()
    monkeypatch.setattr(paged_attention, "_host", s)
    monkeypatch.setattr(device_pages, "_host", s)
    return s


@pytest.mark.parametrize("q", [1, 5])
@pytest.mark.parametrize("scored", [False, True])
@pytest.mark.parametrize("cache", [BF, HF, FP, F8])
def test_the_short_way_and_the_checked_way_agree(spy, cache, scored, q):
    """The same call in one extension step and through Python's checks: same bits."""
    if cache != F8 and not scored:
        pytest.skip("not an extended call")
    g = torch.Generator().manual_seed(3)
    B, Hq, Hkv, D, bs = 3, 8, 2, 64, 16
    dt = BF if cache == F8 else cache
    pool = _random_pool(g, 20, 2, Hkv, bs, D)
    if cache == F8:
        kc, vc, kw = pool.k_layer_view(1), pool.v_layer_view(1), {"key_scales": pool.k_layer_scales(1),
                                                                 "value_scales": pool.v_layer_scales(1)}
    else:
        kc, vc, kw = pool.k_layer_view(1).to(cache), pool.v_layer_view(1).to(cache), {}
    tables = torch.randperm(18, generator=g).reshape(3, 6).int().cuda()
    lens = _i32([0, 17, 70])
    query = torch.randn(B, Hq, q, D, generator=g).to(dt).cuda()
    key, value = (torch.randn(B, q, Hkv, D, generator=g).to(dt).cuda().transpose(1, 2) for _ in range(2))
    slots = (torch.gather(tables.long().cpu(), 1, (lens.cpu()[:, None] + torch.arange(q)) // bs) * bs
             + (lens.cpu()[:, None] + torch.arange(q)) % bs).cuda()
    if scored:
        kw["score_modifiers"] = ScoreModifiers(9.0, 30, torch.rand(Hq, generator=g).cuda(),
                                               _i32([[3] * q, [0] * q, [20] * q])[:, :q], _i32([1, 2, 3]))
    forms = [
        {},
        {"key": key, "value": value},
        {"key": key, "value": value, "slot_mapping": slots.reshape(-1)},
        {"key": key, "value": value, "include": True},
        {"out": torch.empty(B, q, Hq, D, dtype=dt, device="cuda").transpose(1, 2)},
    ]
    paged_attention_decode(query, kc, vc, tables, lens, 0.2, **kw)  # makes workspace and error word
    for form in forms:
        form = dict(form)
        include = form.pop("include", False)
        given = lens + q if include else lens
        states = []
        for validate in (None, True):
            state = [_bits(t).clone() for t in (kc, vc, pool.k_scales, pool.v_scales)]
            del spy.answers[:]
            out = paged_attention_decode(query, kc, vc, tables, given, 0.2, context_lens_include_new=include,
                                         validate=validate, **form, **kw)
            assert spy.answers == ([("decode", True)] if validate is None else []), form.keys()
            if "out" in form:
                assert out is form["out"]
            states.append([out.clone()] + [_bits(t).clone() for t in (kc, vc, pool.k_scales, pool.v_scales)])
            for t, s in zip((kc, vc, pool.k_scales, pool.v_scales), state):
                _bits(t).copy_(s)
        for a, b in zip(*states):
            assert torch.equal(a, b), form.keys()


def test_what_the_short_way_leaves_to_the_checks(spy):
    """Arguments that are converted first, or refused: never launched by the short way."""
    g = torch.Generator().manual_seed(4)
    pool = _random_pool(g, 8, 1, 2, 16, 64)
    kc, vc, ks, vs = pool.k_layer_view(0), pool.v_layer_view(0), pool.k_layer_scales(0), pool.v_layer_scales(0)
    tables, lens = _i32([[0, 1], [2, 3]]), _i32([20, 5])
    query = torch.randn(2, 4, 1, 64, generator=g).to(BF).cuda()

    def call(query=query, tables=tables, lens=lens, ks=ks, vs=vs, **kw):
        return paged_attention_decode(query, kc, vc, tables, lens, 0.125, key_scales=ks, value_scales=vs, **kw)

    want = call()
    rows = torch.zeros(2, 2, 1, 64, dtype=BF, device="cuda")
    del spy.answers[:]
    for same in ({"tables": tables.long()}, {"lens": lens.long()}):  # converted: the same answer
        assert torch.equal(call(**same), want)
    for bad in ({"query": query.float()}, {"query": query[:, :3]}, {"query": query.cpu()}, {"ks": ks[:4]},
                {"vs": vs.double()}, {"vs": None}, {"tables": tables[:1]}, {"lens": lens[:1]}, {"key": rows},
                {"key": rows, "value": rows[:1]}, {"key": rows, "value": rows.half()},
                {"key": rows, "value": rows, "slot_mapping": _i32([1]).long()}, {"out": want.half()},
                {"out": want[:1]}, {"score_modifiers": ScoreModifiers(softcap=-1.0)},
                {"score_modifiers": ScoreModifiers(softcap=1e-40)},
                {"score_modifiers": ScoreModifiers(prefix_lens=_i32([1, 2, 3]))}):
        with pytest.raises((ValueError, RuntimeError)):
            call(**bad)
    assert not any(ok for _, ok in spy.answers)
    del spy.answers[:]
    with pytest.raises((ValueError, RuntimeError)):
        kv_append(rows, rows, kc, vc, _i32([0]).long(), key_scales=ks, value_scales=vs)
    with pytest.raises((ValueError, RuntimeError)):
        copy_pages([kc, ks[:4]], _i32([0]), _i32([1]))
    with pytest.raises((ValueError, RuntimeError)):
        copy_pages([kc], _i32([0, 1]), _i32([1]))
    with pytest.raises(ValueError, match="overlap"):  # one scale of many blocks cannot be appended to
        kv_append(rows, rows, kc, vc, _i32([0, 16]).long(), key_scales=ks[:1].expand(8, 2), value_scales=vs)
    assert spy.answers and not any(ok for _, ok in spy.answers)
    # ... but it can be attended: one scale for a whole cache
    one = torch.full((1, 1), 0.01, device="cuda").expand(8, 2)
    assert torch.equal(call(ks=one, vs=one), call(ks=one.contiguous(), vs=one.contiguous()))


def test_errors_of_a_call_raise_at_the_next():
    g = torch.Generator().manual_seed(5)
    pool = _random_pool(g, 8, 1, 2, 16, 64)
    kc, vc, ks, vs = pool.k_layer_view(0), pool.v_layer_view(0), pool.k_layer_scales(0), pool.v_layer_scales(0)
    query = torch.randn(1, 4, 1, 64, generator=g).to(BF).cuda()
    rows = torch.zeros(2, 2, 1, 64, dtype=BF, device="cuda")

    def attend(table):
        return paged_attention_decode(query, kc, vc, _i32([table]), _i32([20]), 0.125, key_scales=ks, value_scales=vs)

    def append(*slots):
        kv_append(rows, rows, kc, vc, torch.tensor(slots).cuda(), key_scales=ks, value_scales=vs)

    want = attend([1, 2])
    for bad, word in ((lambda: attend([1, 77]), "block"), (lambda: append(3, 4), "two places"),
                      (lambda: append(3, 900), "slot"),
                      (lambda: copy_pages([kc], _i32([0, 0]), _i32([5, 5])), "two places")):
        for following in (lambda: attend([1, 2]), lambda: append(-1, -1), lambda: copy_pages([kc], _i32([-1]), _i32([-1]))):
            bad()
            torch.cuda.synchronize()
            with pytest.raises(IndexError, match=word):
                following()
            following()  # reported once
    assert read_device_errors() == 0
    assert torch.equal(attend([1, 2]), want)


def test_a_pool_written_by_batches_and_copied_on_write():
    """Fp8KVBlockPool beside its plain form: batched writes, then a shared block made
    private by the host allocator before a write lands in it."""
    g = torch.Generator().manual_seed(6)
    bs, H, D = 16, 2, 64
    pool = _random_pool(g, 12, 2, H, bs, D)
    mirror = [c.double().cpu().numpy() if c.dtype == F8 else c.cpu().numpy() for c in pool.caches]

    def write(layer, tables, starts, k, v):
        pool.write_tokens_batch(layer, torch.tensor(tables), torch.tensor(starts), k.cuda(), v.cuda())
        q = k.shape[2]
        slots = [t[(n + i) // bs] * bs + (n + i) % bs for t, n in zip(tables, starts) for i in range(q)]
        for rows, ci, si in ((k, 0, 2), (v, 1, 3)):
            c, s = mirror[ci][:, layer].copy(), mirror[si][:, layer].copy()
            assert append8(rows.float().numpy(), c, s, slots, q, bs) == 0
            mirror[ci][:, layer], mirror[si][:, layer] = c, s
        torch.cuda.synchronize()
        for got, want in zip(pool.caches, mirror):
            assert np.array_equal(got.double().cpu().numpy(), want)

    alloc = BlockRefAllocator(12, bs)
    a = list(alloc.allocate_for_tokens("a", 32).block_ids)
    other = list(alloc.allocate_for_tokens("other", 32).block_ids)
    rows = [torch.randn(2, H, 20, D, generator=g).to(BF) for _ in range(2)]
    for layer in range(2):
        write(layer, [a, other], [0, 5], *rows)
    write(1, [a, other], [20, 25], *(x[:, :, :3] * 8 for x in rows))
    entry = alloc.snapshot_blocks(a)
    b = alloc.allocate_for_tokens("b", 48, borrowed_block_ids=entry)
    pairs = alloc.make_writable("b", 18, 2, pool.copy_blocks)
    assert [old for old, _ in pairs] == [a[1]]
    for c in mirror:
        for old, new in pairs:
            c[new] = c[old]
    write(0, [list(b.block_ids)], [18], *(x[:1, :, :2] * 30 for x in rows))
    with pytest.raises(ValueError):
        pool.copy_blocks([1], [])
    pool.copy_blocks([], [])


@pytest.mark.parametrize("q", [1, 40])
def test_kernels_of_every_kind_share_a_workspace(monkeypatch, q):
    """Rows with CTAs of their own, split rows, balanced rows and the unchanged kernel in
    turn on one workspace: its counters are left as they were found.  (Equal shares of the
    SMs: learned ones move the plain kernel's splits between calls, and with them roundings.)"""
    monkeypatch.setattr(paged_attention, "_SM_SHARES", False)
    g = torch.Generator().manual_seed(7)
    bs, H, D, nb = 16, 8, 128, 4000
    pool = _random_pool(g, nb, 1, H, bs, D)
    kc, vc, ks, vs = pool.k_layer_view(0), pool.v_layer_view(0), pool.k_layer_scales(0), pool.v_layer_scales(0)
    half = [c.to(BF) * 0.01 for c in (kc, vc)]
    cases = []
    for lens in ([30000], [9000, 9000, 200, 5], [300] * 30, [2500] * 24):
        tables = torch.randint(0, nb, (len(lens), (max(lens) + q + bs - 1) // bs), generator=g).int().cuda()
        cases.append((torch.randn(len(lens), 32, q, D, generator=g).to(BF).cuda(), tables, _i32(lens)))

    def all_calls():
        out, kinds = [], set()
        for query, tables, lens in cases:
            out.append(paged_attention_decode(query, kc, vc, tables, lens, 0.08, key_scales=ks, value_scales=vs))
            kinds.add(_lib.last_kernel())
            out.append(paged_attention_decode(query, *half, tables, lens, 0.08))
            kinds.add(_lib.last_kernel())
            out.append(paged_attention_decode(query, *half, tables, lens, 0.08,
                                              score_modifiers=ScoreModifiers(window=4000)))
            kinds.add(_lib.last_kernel())
        return out, kinds

    want, kinds = all_calls()
    assert len(kinds) >= 3, kinds
    for _ in range(3):
        for a, b in zip(want, all_calls()[0]):
            assert torch.equal(a, b)
    assert read_device_errors() == 0


def test_two_streams_with_workspaces_of_their_own():
    g = torch.Generator().manual_seed(8)
    nb, bs = 3000, 16
    pool = _random_pool(g, nb, 1, 8, bs, 128)
    kc, vc, ks, vs = pool.k_layer_view(0), pool.v_layer_view(0), pool.k_layer_scales(0), pool.v_layer_scales(0)
    sets = []
    for lens in ([20000, 15000], [700] * 40):
        tables = torch.randint(0, nb, (len(lens), (max(lens) + bs) // bs), generator=g).int().cuda()
        query = torch.randn(len(lens), 32, 1, 128, generator=g).to(BF).cuda()
        n = _lib.load().pa_decode_workspace_bytes(len(lens), 32, 8, 1, 128, _lib.PA_DTYPE_BFLOAT16, 0)
        sets.append((query, tables, _i32(lens), torch.zeros(n, dtype=torch.uint8, device="cuda"), torch.cuda.Stream()))

    def call(s, **kw):
        return paged_attention_decode(s[0], kc, vc, s[1], s[2], 0.08, key_scales=ks, value_scales=vs,
                                      score_modifiers=ScoreModifiers(softcap=30.0), **kw)

    want = [call(s) for s in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(sets):
            with torch.cuda.stream(s[4]):
                got[i].append(call(s, workspace=s[3]))
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(torch.equal(w, o) for o in outs)


KINDS = [BF, HF, FP, F8]


def _case(cache, lens, q, Hq, Hkv, D, seed, bs=16):
    """(query, kc, vc, tables, lens, scale keywords) with every row's blocks its own."""
    g = torch.Generator().manual_seed(seed)
    n = [(x + q + bs - 1) // bs for x in lens]
    nb, M = sum(n) + 1, max(n)
    perm = torch.randperm(nb, generator=g).int()
    tables = torch.zeros(len(lens), M, dtype=torch.int32)
    at = 0
    for b, k in enumerate(n):
        tables[b, :k] = perm[at: at + k]
        at += k
    dt = BF if cache == F8 else cache
    query = torch.randn(len(lens), Hq, q, D, generator=g).to(dt).cuda()
    kw = {}
    if cache == F8:
        pool = _random_pool(g, nb, 1, Hkv, bs, D)
        kc, vc = pool.k_layer_view(0), pool.v_layer_view(0)
        kw = {"key_scales": pool.k_layer_scales(0), "value_scales": pool.v_layer_scales(0)}
    else:
        kc, vc = (torch.randn(nb, Hkv, bs, D, generator=g).to(dt).cuda() for _ in range(2))
    return query, kc, vc, tables, torch.tensor(lens, dtype=torch.int32), kw


@pytest.mark.parametrize("q,B", [(1, 5), (5, 40), (40, 20)])
@pytest.mark.parametrize("scale", [-0.3, 0.0, 4.0])
@pytest.mark.parametrize("cache", KINDS)
def test_attention_scales_of_any_sign_and_size(cache, scale, q, B):
    query, kc, vc, tables, lens, kw = _case(cache, [3 + 7 * (i % 9) for i in range(B)], q, 16, 8, 64, 11)
    for mods in ((ScoreModifiers(window=20), ScoreModifiers(softcap=3.0)) if cache != F8 else
                 (None, ScoreModifiers(softcap=3.0, window=20))):
        out = paged_attention_decode(query, kc, vc, tables.cuda(), lens.cuda(), scale, score_modifiers=mods,
                                     validate=True, **kw)
        ref, bar = attend64(query, kc, vc, tables, lens, scale, softcap=mods.softcap if mods else 0.0,
                            window=mods.window if mods else 0, **kw)
        check(out, ref, bar)


@pytest.mark.parametrize("q,B", [(1, 5), (1, 200), (40, 20)])
def test_zero_scales(q, B):
    """Blocks of zeros held under a scale of 0: a score of 0, a value of 0; rows of
    nothing but such blocks too."""
    query, kc, vc, tables, lens, kw = _case(F8, [30 + 5 * (i % 7) for i in range(B)], q, 16, 8, 64, 12)
    kw["key_scales"][tables[0, 0].item()] = 0
    kw["value_scales"][tables[1, 0].item()] = 0
    for t in range((35 + q + 16) // 16):
        kw["value_scales"][tables[2, t].item()] = 0
        kw["key_scales"][tables[3, t].item()] = 0
    for mods in (None, ScoreModifiers(window=25)):
        out = paged_attention_decode(query, kc, vc, tables.cuda(), lens.cuda(), 0.125, score_modifiers=mods,
                                     validate=True, **kw)
        ref, bar = attend64(query, kc, vc, tables, lens, 0.125, window=mods.window if mods else 0, **kw)
        check(out, ref, bar)


@pytest.mark.parametrize("q,B", [(1, 3), (1, 200), (40, 20)])
@pytest.mark.parametrize("cache", KINDS)
def test_tables_too_short_for_the_lengths(cache, q, B):
    """Flagged; the other rows are as they should be."""
    query, kc, vc, tables, lens, kw = _case(cache, [20 + i % 5 for i in range(B)], q, 16, 8, 64, 13)
    mods = None if cache == F8 else ScoreModifiers(softcap=9.0)
    long = lens.clone()
    long[1] = 10**6
    args = (query, kc, vc, tables.cuda())
    with pytest.raises(IndexError):
        paged_attention_decode(*args, long.cuda(), 0.125, score_modifiers=mods, validate=True, **kw)
    out = paged_attention_decode(*args, long.cuda(), 0.125, score_modifiers=mods, validate=False, **kw)
    assert read_device_errors() == _lib.PA_DEVERR_TABLE_UNDERRUN
    want = paged_attention_decode(*args, lens.cuda(), 0.125, score_modifiers=mods, validate=True, **kw)
    keep = torch.arange(B) != 1
    ref, bar = attend64(query[keep], kc, vc, tables[keep], lens[keep], 0.125, softcap=mods.softcap if mods else 0.0, **kw)
    check(want[keep], ref, bar)
    check(out[keep], ref, bar)


def test_empty_calls():
    for cache in KINDS:
        query, kc, vc, tables, lens, kw = _case(cache, [5, 9], 1, 8, 2, 64, 14)
        mods = ScoreModifiers(window=3, key_starts=_i32([]))
        for _ in range(2):
            out = paged_attention_decode(query[:0], kc, vc, tables[:0].cuda(), lens[:0].cuda(), 0.125,
                                         score_modifiers=mods, **kw)
            assert out.shape == (0, 8, 1, 64)
        if cache == F8:
            none = torch.zeros(0, 2, 1, 64, device="cuda")
            kv_append(none, none, kc, vc, torch.zeros(0, dtype=torch.int64, device="cuda"), **kw)
    pages = DevicePages(4, 16, 4, 4)
    for _ in range(2):
        pages.free(_i32([]))
        pages.fork(_i32([]), _i32([]))
        pages.reserve(_i32([]), _i32([]))
    assert pages.read_errors() == 0 and read_device_errors() == 0


@pytest.mark.parametrize("cache", KINDS)
def test_errors_of_every_part_of_a_call_are_reported(cache):
    """The append of a changed-score call, and the halves of a batch beyond one launch."""
    query, kc, vc, tables, lens, kw = _case(cache, [5, 9], 1, 8, 2, 64, 15)
    kw["score_modifiers"] = ScoreModifiers(window=30)
    rows = torch.zeros(2, 2, 1, 64, dtype=query.dtype, device="cuda")
    args = (query, kc, vc, tables.cuda(), lens.cuda(), 0.125)
    bad = dict(key=rows, value=rows, slot_mapping=torch.tensor([10**6, -1]).cuda())
    with pytest.raises(IndexError, match="slot"):
        paged_attention_decode(*args, validate=True, **bad, **kw)
    for how in ({}, {"out": torch.empty_like(query)}, {"validate": False}):
        paged_attention_decode(*args, **bad, **how, **kw)
        torch.cuda.synchronize()
        with pytest.raises(IndexError, match="slot"):
            paged_attention_decode(*args, **kw)
    B = 9000
    many = torch.zeros(B, 1, dtype=torch.int32, device="cuda")
    many[B - 1] = 10**6
    big = (query[:1].expand(B, 8, 1, 64).contiguous(), kc, vc, many, torch.full((B,), 3, dtype=torch.int32).cuda(), 0.125)
    with pytest.raises(IndexError, match="block"):
        paged_attention_decode(*big, validate=True, **kw)
    paged_attention_decode(*big, **kw)
    torch.cuda.synchronize()
    with pytest.raises(IndexError, match="block"):
        paged_attention_decode(*big, **kw)
    assert read_device_errors() == 0
