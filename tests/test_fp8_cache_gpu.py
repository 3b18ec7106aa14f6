"""Caches held in 8 bits: the append against its definition bit for bit, attention
over them against 64 bits."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from _ops64 import F8, append8, attend64, check
from llm_serving_runtime_b200 import _lib, kv_append, paged_attention_decode, read_device_errors
from llm_serving_runtime_b200.cuda_graph import DecodeStepGraph

pytestmark = pytest.mark.gpu
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _cache(nb, H, bs, D, g, *, spread=2, pow2=True, layers=1):
    """(codes, scales) on the GPU as layer views of pools, random."""
    codes = (torch.randn(nb, layers, H, bs, D, generator=g) * 100).clamp(-448, 448).to(F8)
    scales = torch.exp2(torch.randint(-8 - spread, -7 + spread, (nb, layers, H), generator=g).float())
    if not pow2:
        scales *= 1 + torch.rand(scales.shape, generator=g)
    return codes.cuda()[:, layers - 1], scales.cuda()[:, layers - 1]


def _tables(lens, q, bs, g, extra=2):
    n = [(int(x) + q + bs - 1) // bs for x in lens]
    nb = sum(n) + extra
    perm = torch.randperm(nb, generator=g).int()
    bt = torch.zeros(len(n), max(max(n), 1), dtype=torch.int32)
    at = 0
    for b, k in enumerate(n):
        bt[b, :k] = perm[at: at + k]
        at += k
    return bt, nb


def _slots(bt, lens, q, bs):
    pos = torch.as_tensor(lens)[:, None] + torch.arange(q)
    return (torch.gather(bt.long(), 1, pos // bs) * bs + pos % bs).reshape(-1)


class Append:
    """One cache on the GPU beside its plain form."""

    def __init__(self, nb, H, bs, D, seed, **kw):
        g = _gen(seed)
        self.bs = bs
        self.gpu = [x for _ in range(2) for x in _cache(nb, H, bs, D, g, **kw)]  # kc, ks, vc, vs
        self.cpu = [x.double().cpu().numpy().copy() if x.dtype == F8 else x.cpu().numpy().copy() for x in self.gpu]

    def append(self, key, value, slots, *, q, flags=0, **form):
        want = 0
        for i, rows in enumerate((key, value)):
            want |= append8(rows.float().numpy(), self.cpu[2 * i], self.cpu[2 * i + 1], slots, q, self.bs)
        if form:
            kv_append(key.cuda(), value.cuda(), self.gpu[0], self.gpu[2], key_scales=self.gpu[1],
                      value_scales=self.gpu[3], validate=False, **form)
        else:
            kv_append(key.cuda(), value.cuda(), self.gpu[0], self.gpu[2], slots.cuda(), key_scales=self.gpu[1],
                      value_scales=self.gpu[3], validate=False)
        assert read_device_errors() == flags == want
        self.same()

    def same(self):
        for got, want in zip(self.gpu, self.cpu):
            got = got.double().cpu().numpy()
            assert np.array_equal(got, want, equal_nan=True), np.argwhere(got != want)[:4]


def _rows(B, H, q, D, g, dtype, size=1.0):
    mul = torch.exp2(torch.randint(-3, 4, (B, H, q, 1), generator=g).float()) * size
    return (torch.randn(B, H, q, D, generator=g) * mul).to(dtype)


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("H,D,bs", [(2, 64, 16), (8, 128, 16), (1, 16, 8), (3, 96, 32), (4, 128, 256)])
@pytest.mark.parametrize("q", [1, 7, 70])
def test_append_through_tables(dtype, H, D, bs, q):
    g = _gen(H * D + bs + q)
    lens = torch.randint(0, 3 * bs, (5,), generator=g)
    lens[0], lens[1] = 0, bs  # fresh blocks
    bt, nb = _tables(lens, q, bs, g)
    c = Append(nb, H, bs, D, q, layers=2)
    k, v = _rows(5, H, q, D, g, dtype), _rows(5, H, q, D, g, dtype, 5.0)
    c.append(k, v, _slots(bt, lens, q, bs), q=q, block_tables=bt.cuda(), positions=lens.cuda())


@pytest.mark.parametrize("q", [1, 5, 33])
def test_append_through_slots_with_padding(q):
    g = _gen(q)
    lens = torch.randint(0, 100, (6,), generator=g)
    bt, nb = _tables(lens, q, 16, g)
    slots = _slots(bt, lens, q, 16)
    slots[torch.rand(slots.shape, generator=g) < 0.2] = -1
    c = Append(nb, 2, 16, 64, q)
    c.append(_rows(6, 2, q, 64, g, BF), _rows(6, 2, q, 64, g, BF), slots, q=q)


def test_a_sequence_grows_token_by_token():
    """Every token re-rounds the block where it raises its scale, as the definition says."""
    g = _gen(3)
    c = Append(4, 2, 16, 32, 3)
    bt = torch.tensor([[2, 0, 3]], dtype=torch.int32)
    for t in range(40):
        size = 2.0 ** (t % 7 - 3)
        c.append(_rows(1, 2, 1, 32, g, BF, size), _rows(1, 2, 1, 32, g, BF, 1 / size), _slots(bt, [t], 1, 16), q=1,
                 block_tables=bt.cuda(), positions=torch.tensor([t]).cuda())


def test_a_scale_that_is_no_power_of_two():
    g = _gen(4)
    lens = [5, 20, 9]
    bt, nb = _tables(lens, 4, 16, g)
    c = Append(nb, 2, 16, 64, 4, pow2=False)
    c.append(_rows(3, 2, 4, 64, g, BF, 0.01), _rows(3, 2, 4, 64, g, BF, 50.0), _slots(bt, lens, 4, 16), q=4)


@pytest.mark.parametrize("offset", [0, 3])
def test_values_at_the_types_ends(offset):
    """0, infinities, NaN, the largest and least values, a bad held scale."""
    c = Append(6, 1, 8, 16, 5)
    for i, s in enumerate((0.0, float("nan"), float("inf"), -1.0)):
        c.gpu[1][i, 0] = s
        c.cpu[1][i, 0] = s
    rows = torch.zeros(6, 1, 1, 16)
    rows[0, 0, 0, 0] = float("inf")
    rows[1, 0, 0, :3] = torch.tensor([float("nan"), float("-inf"), 2.5])
    rows[2, 0, 0, :2] = torch.tensor([3.3e38, -1.0])
    rows[3, 0, 0, :2] = torch.tensor([1e-38, -1e-45])
    rows[4, 0, 0, 0] = 448.0 * 2.0**-9
    slots = torch.arange(6) * 8 + offset
    c.append(rows, rows, slots, q=1)


def test_long_padding_between_a_blocks_tokens():
    """Padding of any length neither ends a run nor hides the slot before it."""
    g = _gen(60)
    q = 9000
    slots = torch.full((2 * q,), -1, dtype=torch.int64)
    slots[0], slots[4000], slots[4001], slots[8999] = 5, 6, 16, 17
    slots[q + 8500], slots[q + 8999] = 40, 41
    c = Append(4, 1, 16, 16, 60)
    rows = torch.zeros(2, 1, q, 16)
    for i in (0, 4000, 4001, 8500, 8999):
        rows[:, :, i] = torch.randn(2, 1, 16, generator=g) * 2.0 ** (i % 3)
    c.append(rows.to(BF), rows.to(BF), slots, q=q)


@pytest.mark.parametrize("H", [1, 5])
@pytest.mark.parametrize("clash", [False, True])
def test_many_runs_among_neighbouring_tokens(H, clash):
    """Slots in any order: runs of one to three tokens, padding between them, two rows;
    with a block that the row, or the other row, comes back to."""
    g = _gen(62)
    bs, q = 16, 75
    blocks = torch.randperm(200, generator=g).tolist()
    slots = torch.full((2, q), -1, dtype=torch.int64)
    for b in range(2):
        t = 0
        while t < q:
            blk = blocks.pop()
            for o in torch.randperm(bs, generator=g)[: 1 + t % 3].tolist():
                if t < q and t % 7 != 5:
                    slots[b, t] = blk * bs + o
                t += 1
    if clash:
        slots[0, 60] = slots[0, 2] // bs * bs + 9
        slots[1, 30] = slots[0, 20]
    c = Append(200, H, bs, 32, 62)
    k, v = _rows(2, H, q, 32, g, BF), _rows(2, H, q, 32, g, BF)
    c.append(k, v, slots.reshape(-1), q=q, flags=_lib.PA_DEVERR_BLOCK_CONFLICT if clash else 0)


def test_a_slot_given_twice_takes_the_last_token():
    g = _gen(6)
    c = Append(4, 2, 16, 64, 6)
    slots = torch.tensor([16, 17, 17, 16, -1, 17, 35, 35])
    c.append(_rows(1, 2, 8, 64, g, HF), _rows(1, 2, 8, 64, g, HF), slots, q=8)


def test_two_rows_in_one_block_are_refused():
    g = _gen(7)
    c = Append(6, 2, 16, 64, 7)
    k, v = _rows(3, 2, 2, 64, g, BF), _rows(3, 2, 2, 64, g, BF)
    c.append(k, v, torch.tensor([16, 17, 18, 19, 80, 81]), q=2, flags=0x40)
    c.append(k, v, torch.tensor([16, 32, 20, 21, 33, 34]), q=2, flags=0x40)
    bt = torch.tensor([[1, 2], [3, 1], [4, 5]], dtype=torch.int32)
    lens = torch.tensor([3, 20, 16])
    c.append(k, v, _slots(bt, lens, 2, 16), q=2, flags=0x40, block_tables=bt.cuda(), positions=lens.cuda())


def test_bad_slots_blocks_and_positions_are_skipped():
    g = _gen(8)
    c = Append(4, 2, 16, 64, 8)
    k, v = _rows(2, 2, 1, 64, g, BF), _rows(2, 2, 1, 64, g, BF)
    c.append(k, v, torch.tensor([64, 5]), q=1, flags=0x4)
    for bt, lens, flag in (([[4], [0]], [3, 3], 0x1), ([[-1], [0]], [3, 3], 0x1), ([[0], [1]], [16, 3], 0x2),
                           ([[0], [1]], [-1, 3], 0x4)):
        ok = torch.tensor([-1, _slots(torch.tensor(bt), [0, 3], 1, 16)[1]])
        bt, lens = torch.tensor(bt, dtype=torch.int32), torch.tensor(lens)
        for i, rows in enumerate((k, v)):
            append8(rows.float().numpy(), c.cpu[2 * i], c.cpu[2 * i + 1], ok, 1, 16)
        with pytest.raises(IndexError):
            kv_append(k.cuda(), v.cuda(), c.gpu[0], c.gpu[2], block_tables=bt.cuda(), positions=lens.cuda(),
                      key_scales=c.gpu[1], value_scales=c.gpu[3], validate=True)
        c.same()


def test_a_row_that_starts_before_zero_writes_the_rest():
    g = _gen(9)
    c = Append(3, 2, 16, 64, 9)
    k, v = _rows(1, 2, 5, 64, g, BF), _rows(1, 2, 5, 64, g, BF)
    slots = torch.tensor([-1, -1, 16, 17, 18])
    for i, rows in enumerate((k, v)):
        append8(rows.float().numpy(), c.cpu[2 * i], c.cpu[2 * i + 1], slots, 5, 16)
    kv_append(k.cuda(), v.cuda(), c.gpu[0], c.gpu[2], block_tables=torch.tensor([[1, 2]], dtype=torch.int32).cuda(),
              positions=torch.tensor([-2]).cuda(), key_scales=c.gpu[1], value_scales=c.gpu[3], validate=False)
    assert read_device_errors() == 0x4
    c.same()


def test_strided_and_unaligned_rows():
    g = _gen(10)
    lens = [4, 30]
    bt, nb = _tables(lens, 3, 16, g)
    slots = _slots(bt, lens, 3, 16)
    for cut in (slice(0, 64), slice(1, 65), slice(2, 66)):
        c = Append(nb, 2, 16, 64, 10)
        big = _rows(2, 3, 2, 70, g, HF)  # [B, q, H, D'] as projections give them
        k, v = big[..., cut].transpose(1, 2), (big * 2)[..., cut].transpose(1, 2)
        for i, rows in enumerate((k, v)):
            append8(rows.float().numpy(), c.cpu[2 * i], c.cpu[2 * i + 1], slots, 3, 16)
        bg, b2 = big.cuda(), (big * 2).cuda()
        kv_append(bg[..., cut].transpose(1, 2), b2[..., cut].transpose(1, 2), c.gpu[0], c.gpu[2], slots.cuda(),
                  key_scales=c.gpu[1], value_scales=c.gpu[3], validate=True)
        c.same()


# ---- attention -----------------------------------------------------------------------

def _attend(dtype, lens, q, Hq, Hkv, D, bs, *, seed=0, pow2=True, size=1.0, tweak=None, kernel=None, include=False,
            scores=None, spread=2):
    g = _gen(seed)
    bt, nb = _tables(lens, q, bs, g)
    kc, ks = _cache(nb, Hkv, bs, D, g, pow2=pow2, layers=2, spread=spread)
    vc, vs = _cache(nb, Hkv, bs, D, g, pow2=pow2, layers=2, spread=spread)
    query = (torch.randn(len(lens), Hq, q, D, generator=g) * size).to(dtype).cuda()
    lens = torch.tensor(lens, dtype=torch.int32)
    if tweak:
        tweak(query, kc, vc, ks, vs, bt)
    given = (lens + q if include else lens).cuda()
    out = paged_attention_decode(query, kc, vc, bt.cuda(), given, D**-0.5, key_scales=ks, value_scales=vs,
                                 validate=True, context_lens_include_new=include)
    if kernel:
        assert _lib.last_kernel() == kernel
    ref, bar = attend64(query, kc, vc, bt, lens, D**-0.5, key_scales=ks, value_scales=vs)
    check(out, ref, bar)
    return out


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("Hq,Hkv,D", [(32, 8, 128), (14, 2, 64), (8, 8, 64), (12, 4, 96), (16, 1, 128), (8, 2, 32),
                                      (4, 2, 16), (40, 2, 112)])
def test_decode(dtype, Hq, Hkv, D):
    _attend(dtype, [0, 1, 15, 16, 17, 130, 700], 1, Hq, Hkv, D, 16, seed=D)


@pytest.mark.parametrize("bs", [8, 16, 32, 64, 256])
@pytest.mark.parametrize("q", [1, 4])
def test_block_sizes(bs, q):
    _attend(BF, [0, 3, 9, 250, 513], q, 8, 2, 128, bs, seed=bs)
    _attend(HF, [1, 7, 8, 255], q, 8, 4, 64, bs, seed=bs + 1, pow2=False)


def test_a_long_row_split_over_the_gpu():
    _attend(BF, [20011], 1, 8, 2, 128, 16, seed=1)
    _attend(HF, [9000, 5], 3, 4, 1, 64, 16, seed=2)


def test_many_ragged_rows():
    g = _gen(5)
    _attend(BF, torch.randint(0, 600, (70,), generator=g).tolist(), 1, 8, 2, 128, 16, seed=5)


def test_lengths_that_include_the_new_tokens_and_empty_rows():
    _attend(BF, [-1, 40], 1, 8, 2, 64, 16, seed=6, include=True)
    out = _attend(HF, [-3, 0, 2], 3, 8, 2, 64, 16, seed=7, include=True)
    assert bool((out[0] == 0).all())


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D,bs", [(128, 16), (64, 8), (96, 32)])
def test_multi_query(dtype, D, bs):
    _attend(dtype, [0, 5, 70, 33] * 5, 33, 16, 8, D, bs, seed=D, kernel="pa::prefill_mma_kernel<ext>")


def test_queries_of_any_size():
    """bf16 rows beyond fp16's range, and rows of tiny and of zero elements."""
    def tweak(query, *_):
        query[0] *= 1e30
        query[1] *= 1e-30
        query[2, :, :, 3:] = 0
        query[3] = 0
    def quiet(query, kc, vc, ks, vs, bt):
        tweak(query)
        ks *= 1e-30
        ks[bt[1:].long().cuda()] *= 1e30
    _attend(BF, [30, 31, 50, 7], 1, 8, 2, 64, 16, seed=8, tweak=quiet)


def test_blocks_of_very_different_scale():
    """A block of huge values and no weight leaves the others' digits alone."""
    def tweak(query, kc, vc, ks, vs, bt):
        vs[bt[0, 1].long()] *= 2.0**40  # huge values ...
        kc.view(torch.uint8)[bt[0, 1].long()] = 0x7e  # ... under scores far below the rest
        query[0] = -query[0].abs()
        vs[bt[1, 0].long()] = 0  # zeros, and a zero scale
        vs[bt[2, 2].long()] *= 2.0**-40
    _attend(BF, [60, 60, 60], 1, 8, 2, 64, 16, seed=9, tweak=tweak)


def test_nan_in_places_a_row_does_not_see():
    """Behind a row's end, and in later tokens of the same step."""
    def tweak(query, kc, vc, ks, vs, bt):
        # row 0: 3 tokens of its last block are attended, the rest holds NaN codes
        for c in (kc, vc):
            c.view(torch.uint8)[bt[0, 1].long(), :, 3:] = 0x7f
            c.view(torch.uint8)[bt[1, 0].long(), :, 11] = 0xff  # the third of four new tokens
    out = _attend(HF, [15, 9, 40], 4, 8, 2, 64, 16, seed=10, tweak=tweak)
    assert bool(torch.isnan(out[1, :, 2:]).all()) and not bool(torch.isnan(out[1, :, :2]).any())
    assert not bool(torch.isnan(out[0]).any())


def test_nan_scales_stay_in_their_head():
    def tweak(query, kc, vc, ks, vs, bt):
        ks[bt[0, 0].long(), 0] = float("nan")
        vs[bt[1, 1].long(), 1] = float("nan")
    out = _attend(BF, [30, 30, 30], 1, 8, 2, 64, 16, seed=11, tweak=tweak)
    assert bool(torch.isnan(out[0, :4]).all()) and not bool(torch.isnan(out[0, 4:]).any())
    assert bool(torch.isnan(out[1, 4:]).all()) and not bool(torch.isnan(out[1, :4]).any())


def test_bad_block_ids_raise_and_do_not_read():
    g = _gen(12)
    kc, ks = _cache(4, 2, 16, 64, g)
    q = torch.randn(2, 4, 1, 64, generator=g).to(BF).cuda()
    for bad in (4, -1, 2**31 - 1):
        bt = torch.tensor([[bad, 1], [2, 3]], dtype=torch.int32).cuda()
        with pytest.raises(IndexError, match="out of range"):
            paged_attention_decode(q, kc, kc, bt, torch.tensor([20, 20]).cuda(), 0.125, key_scales=ks, value_scales=ks,
                                   validate=True)


def test_the_step_append_and_attend_with_a_graph():
    """Steps through the public call, eagerly and as a replayed graph, agree."""
    g = _gen(13)
    B, Hq, Hkv, D, bs = 3, 8, 2, 64, 16
    lens0 = [0, 17, 30]
    bt, nb = _tables([x + 12 for x in lens0], 1, bs, g)
    layers = [_cache(nb, Hkv, bs, D, g) + _cache(nb, Hkv, bs, D, g) for _ in range(2)]
    eager = [[t.clone() for t in layer] for layer in layers]
    graph = DecodeStepGraph([x[0] for x in layers], [x[2] for x in layers], batch=B, max_blocks=bt.shape[1],
                            num_q_heads=Hq, scale=D**-0.5, dtype=BF, key_scales=[x[1] for x in layers],
                            value_scales=[x[3] for x in layers])
    for step in range(6):
        lens = torch.tensor([x + step for x in lens0], dtype=torch.int32)
        slots = _slots(bt, lens.long(), 1, bs).cuda()
        qs, ks, vs = ([_rows(B, H, 1, D, g, BF).cuda() for _ in layers] for H in (Hq, Hkv, Hkv))
        got = graph.step(block_tables=bt.cuda(), context_lens=lens.cuda(), slot_mapping=slots, queries=qs, new_keys=ks,
                         new_values=vs)
        for i, layer in enumerate(eager):
            out = paged_attention_decode(qs[i], layer[0], layer[2], bt.cuda(), lens.cuda(), D**-0.5, slots, ks[i],
                                         vs[i], key_scales=layer[1], value_scales=layer[3], validate=True)
            assert torch.equal(out, got[i])
            for a, b in zip(layer, layers[i]):
                assert torch.equal(a.view(torch.uint8) if a.dtype == F8 else a,
                                   b.view(torch.uint8) if b.dtype == F8 else b)
            ref, bar = attend64(qs[i], layer[0], layer[2], bt, lens, D**-0.5, key_scales=layer[1],
                                value_scales=layer[3])
            check(out, ref, bar)


def test_batches_beyond_the_shared_memory_tables():
    g = _gen(14)
    B = 9000
    kc, ks = _cache(40, 1, 16, 64, g)
    bt = torch.randint(0, 40, (B, 2), generator=g).int()
    lens = torch.randint(0, 30, (B,), generator=g).int()
    q = torch.randn(B, 2, 1, 64, generator=g).to(BF).cuda()
    out = paged_attention_decode(q, kc, kc, bt.cuda(), lens.cuda(), 0.125, key_scales=ks, value_scales=ks, validate=True)
    rows = [0, 4499, 4500, 8999]
    ref, bar = attend64(q[rows], kc, kc, bt[rows], lens[rows], 0.125, key_scales=ks, value_scales=ks)
    check(out[rows], ref, bar)


def test_caches_past_32_bit_offsets():
    """Codes beyond 2^32 bytes: appended to and attended at both ends."""
    g = _gen(61)
    nb, H, bs, D = 2_200_000, 1, 16, 128
    codes = torch.zeros(nb, H, bs, D, dtype=torch.uint8, device="cuda").view(F8)
    scales = torch.zeros(nb, H, device="cuda")
    bt = torch.tensor([[nb - 1, 3], [nb - 7, nb - 2]], dtype=torch.int32)
    k = _rows(2, 1, 20, D, g, BF).cuda()
    zero = torch.zeros(2, dtype=torch.int32, device="cuda")
    kv_append(k, k, codes, codes, block_tables=bt.cuda(), positions=zero, key_scales=scales, value_scales=scales,
              validate=True)
    q = torch.randn(2, 4, 1, D, generator=g).to(BF).cuda()
    lens = torch.tensor([19, 19], dtype=torch.int32)
    out = paged_attention_decode(q, codes, codes, bt.cuda(), lens.cuda(), D**-0.5, key_scales=scales,
                                 value_scales=scales, validate=True)
    ids = bt.long().reshape(-1)
    small = torch.arange(4, dtype=torch.int32).reshape(2, 2)
    c = codes.view(torch.uint8)[ids.cuda()].view(F8)
    ref, bar = attend64(q, c, c, small, lens, D**-0.5, key_scales=scales[ids.cuda()], value_scales=scales[ids.cuda()])
    check(out, ref, bar)
    want = k[1, 0, :16].float()
    got = codes.view(torch.uint8)[nb - 7, 0].view(F8).float() * scales[nb - 7, 0]
    # a code is off by half a step of its value, or of the least normal one
    assert bool(((got - want).abs() <= want.abs() * 2.0**-4 + scales[nb - 7, 0] * 2.0**-10).all())


def test_refusals():
    g = _gen(15)
    kc, ks = _cache(4, 2, 16, 64, g)
    q = torch.zeros(1, 4, 1, 64, dtype=BF, device="cuda")
    bt, lens = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.tensor([3]).cuda()
    half = torch.zeros(4, 2, 16, 64, dtype=BF, device="cuda")

    def call(query=q, k=kc, v=kc, **kw):
        paged_attention_decode(query, k, v, bt, lens, 0.125, **kw)

    with pytest.raises(ValueError, match="needs key_scales"):
        call()
    with pytest.raises(ValueError, match="belong to"):
        call(k=half, v=half, key_scales=ks, value_scales=ks)
    with pytest.raises(ValueError, match="fp16 or bf16"):
        call(query=q.float(), key_scales=ks, value_scales=ks)
    with pytest.raises(ValueError, match="num_kv_heads"):
        call(key_scales=ks[:, :1], value_scales=ks)
    with pytest.raises(ValueError, match="float32"):
        call(key_scales=ks.half(), value_scales=ks)
    with pytest.raises(ValueError, match="multiple of 16"):
        paged_attention_decode(q[..., :56].contiguous(), kc[..., :56], kc[..., :56], bt, lens, 0.125, key_scales=ks,
                               value_scales=ks)
    rows = torch.zeros(1, 2, 1, 64, device="cuda")
    with pytest.raises(ValueError, match="same dtype"):
        kv_append(rows, rows.half(), kc, kc, torch.tensor([0]).cuda(), key_scales=ks, value_scales=ks)
    with pytest.raises(ValueError, match="fp32, fp16 or bf16"):
        kv_append(rows.double(), rows.double(), kc, kc, torch.tensor([0]).cuda(), key_scales=ks, value_scales=ks)
