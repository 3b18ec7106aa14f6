"""Capped, biased and masked scores against the definition in 64 bits."""

from __future__ import annotations

import pytest
import torch

from _ops64 import F8, attend64, check
from llm_serving_runtime_b200 import ScoreModifiers, _lib, paged_attention_decode, read_device_errors
from llm_serving_runtime_b200.cuda_graph import DecodeStepGraph
from llm_serving_runtime_b200.prefix_sharing import PrefixGroups

pytestmark = pytest.mark.gpu
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
FP8 = "fp8"  # an 8-bit cache under bf16 queries


def _setup(dtype, lens, q, Hq, Hkv, D, bs, seed, size=1.0):
    g = torch.Generator().manual_seed(seed)
    n = [(max(int(x), 0) + q + bs - 1) // bs for x in lens]
    nb = sum(n) + 2
    perm = torch.randperm(nb, generator=g).int()
    bt = torch.zeros(len(n), max(max(n), 1), dtype=torch.int32)
    at = 0
    for b, k in enumerate(n):
        bt[b, :k] = perm[at: at + k]
        at += k
    ks = vs = None
    x = [torch.randn(nb, 2, Hkv, bs, D, generator=g) for _ in range(2)]
    if dtype == FP8:
        ks, vs = (torch.exp2(torch.randint(-9, -5, (nb, Hkv), generator=g).float()).cuda() for _ in range(2))
        kc, vc = ((c[:, 1] * 100).clamp(-448, 448).to(F8).cuda() for c in x)
        dtype = BF
    else:
        kc, vc = (c.to(dtype).cuda()[:, 1] for c in x)
    query = (torch.randn(len(lens), Hq, q, D, generator=g) * size).to(dtype).cuda()
    return query, kc, vc, bt, torch.tensor(lens, dtype=torch.int32), ks, vs


def _run(s, mods, *, kernel=None, validate=True, include=False):
    query, kc, vc, bt, lens, ks, vs = s
    scale = query.shape[-1] ** -0.5
    given = (lens + query.shape[2] if include else lens).cuda()
    out = paged_attention_decode(query, kc, vc, bt.cuda(), given, scale, key_scales=ks, value_scales=vs,
                                 score_modifiers=mods, validate=validate, context_lens_include_new=include)
    if kernel:
        assert _lib.last_kernel() == kernel
    ref, bar = attend64(query, kc, vc, bt, lens, scale, key_scales=ks, value_scales=vs, softcap=mods.softcap,
                        window=mods.window, alibi_slopes=mods.alibi_slopes, key_starts=mods.key_starts,
                        prefix_lens=mods.prefix_lens)
    check(out, ref, bar)
    return out


def _slopes(Hq):
    return torch.exp2(-8.0 * torch.arange(1, Hq + 1).float() / Hq).cuda()


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _starts(lens, q, every):
    pos = torch.tensor(lens)[:, None] + torch.arange(q)
    return (pos // every * every).int().cuda()


LENS = [0, 1, 14, 15, 16, 17, 100, 333]


def _mods(kind, lens, q, Hq):
    return {
        "cap": ScoreModifiers(softcap=5.0),
        "large cap": ScoreModifiers(softcap=1e4),
        "window": ScoreModifiers(window=20),
        "window of 1": ScoreModifiers(window=1),
        "window of all": ScoreModifiers(window=2**31 - 1),
        "bias": ScoreModifiers(alibi_slopes=_slopes(Hq)),
        "documents": ScoreModifiers(key_starts=_starts(lens, q, 50)),
        "starts of rows": ScoreModifiers(key_starts=_i32([x // 2 for x in lens])),
        "prefix": ScoreModifiers(prefix_lens=_i32([(7 * i) % 40 for i in range(len(lens))])),
        "none": ScoreModifiers(),
        "all": ScoreModifiers(softcap=20.0, window=40, alibi_slopes=_slopes(Hq), key_starts=_starts(lens, q, 30),
                              prefix_lens=_i32([5] * len(lens))),
    }[kind]


KINDS = ["cap", "large cap", "window", "window of 1", "window of all", "bias", "documents", "starts of rows", "prefix",
         "none", "all"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [BF, HF, FP, FP8])
def test_single_tokens(dtype, kind):
    _run(_setup(dtype, LENS, 1, 8, 2, 64, 16, 1, 2.0), _mods(kind, LENS, 1, 8))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [BF, FP, FP8])
def test_several_tokens(dtype, kind):
    _run(_setup(dtype, LENS, 5, 16, 4, 128, 16, 2, 2.0), _mods(kind, LENS, 5, 16))


@pytest.mark.parametrize("kind", ["cap", "window", "bias", "documents", "prefix", "all"])
@pytest.mark.parametrize("dtype,D,bs", [(BF, 128, 16), (HF, 64, 8), (FP8, 128, 32), (FP8, 64, 8)])
def test_chunks(dtype, D, bs, kind):
    lens = [0, 40, 97, 16, 3] * 4
    kernel = "pa::prefill_mma_kernel<ext>" if dtype == FP8 else "pa::prefill_umma_kernel<scored>"
    _run(_setup(dtype, lens, 37, 16, 8, D, bs, 3), _mods(kind, lens, 37, 16), kernel=kernel)


@pytest.mark.parametrize("kind", ["all", "documents", "window"])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_chunks_of_unaligned_rows(dtype, kind):
    """Query rows that are not 16-byte aligned go to the mma.sync kernel."""
    lens = [0, 40, 97, 16, 3] * 4
    s = list(_setup(dtype, lens, 37, 16, 8, 64, 16, 3))
    wide = torch.zeros(20, 16, 37, 66, dtype=dtype, device="cuda")
    wide[..., 2:] = s[0]
    s[0] = wide[..., 2:]
    _run(s, _mods(kind, lens, 37, 16), kernel="pa::prefill_mma_kernel<ext>")


@pytest.mark.parametrize("dtype", [BF, HF])
def test_long_chunks(dtype):
    """Several row blocks and chunks a sequence; documents, windows and a prefix across them."""
    lens = [5, 300, 130, 700, 64, 0, 411]
    s = _setup(dtype, lens, 150, 16, 8, 64, 16, 30)
    _run(s, ScoreModifiers(key_starts=_starts(lens, 150, 110), softcap=8.0), kernel="pa::prefill_umma_kernel<scored>")
    _run(s, ScoreModifiers(window=70, alibi_slopes=_slopes(16)), kernel="pa::prefill_umma_kernel<scored>")
    _run(s, ScoreModifiers(prefix_lens=_i32([333] * 7)), kernel="pa::prefill_umma_kernel<scored>")


@pytest.mark.parametrize("Hq,Hkv,D,bs", [(14, 2, 64, 16), (4, 4, 96, 8), (16, 1, 128, 64), (8, 2, 32, 256), (6, 3, 80, 32)])
@pytest.mark.parametrize("dtype", [BF, HF, FP, FP8])
def test_heads_and_blocks(dtype, Hq, Hkv, D, bs):
    lens = [3, 70, 600]
    _run(_setup(dtype, lens, 2, Hq, Hkv, D, bs, 4), _mods("all", lens, 2, Hq))
    _run(_setup(dtype, lens, 1, Hq, Hkv, D, bs, 5), ScoreModifiers(window=33, softcap=3.0))


@pytest.mark.parametrize("dtype", [BF, FP, FP8])
def test_a_long_row(dtype):
    """Split over the GPU, with and without a window; a long document."""
    s = _setup(dtype, [12007], 1, 8, 2, 64, 16, 6)
    _run(s, ScoreModifiers(window=5000, softcap=30.0))
    _run(s, ScoreModifiers(alibi_slopes=_slopes(8) * 0.01))
    _run(s, ScoreModifiers(key_starts=_i32([11990])))


@pytest.mark.parametrize("dtype", [BF, HF, FP, FP8])
@pytest.mark.parametrize("q", [1, 3, 40])
def test_rows_that_see_nothing(dtype, q):
    """Documents that start behind the token, alone, beside others and in all rows."""
    lens = [20, 50, 5] * 7
    s = _setup(dtype, lens, q, 16, 8, 64, 16, 7)
    starts = _starts(lens, q, 10**6)
    starts[0] = 10**6
    starts[1, q // 2] = 2**31 - 1
    starts[4, 0] = lens[4] + 1
    out = _run(s, ScoreModifiers(key_starts=starts))
    assert bool((out[0] == 0).all()) and bool((out[1, :, q // 2] == 0).all())
    out = _run(s, ScoreModifiers(key_starts=torch.full_like(starts, 10**6)))
    assert bool((out == 0).all())


@pytest.mark.parametrize("dtype", [BF, HF, FP, FP8])
def test_negative_starts_and_prefixes_and_short_rows(dtype):
    s = _setup(dtype, [-2, 0, 30], 4, 8, 2, 64, 16, 8)
    _run(s, ScoreModifiers(key_starts=_i32([-5, -1, -(2**31)]), prefix_lens=_i32([9, -3, 2**31 - 1])), include=True)


@pytest.mark.parametrize("dtype", [BF, HF, FP, FP8])
@pytest.mark.parametrize("q", [4, 40])
def test_the_widest_window_over_rows_shorter_than_the_call(dtype, q):
    """Tokens before the sequence's start see nothing, the others everything."""
    s = _setup(dtype, [-3 * q // 4, -q // 2, -1, -q, 30], q, 8, 2, 64, 16, 18)
    _run(s, ScoreModifiers(window=2**31 - 1, prefix_lens=_i32([2, 0, 1, 3, 9])), include=True)


@pytest.mark.parametrize("dtype", [BF, HF, FP, FP8])
@pytest.mark.parametrize("q", [1, 4, 40])
def test_what_is_hidden_may_be_anything(dtype, q):
    """NaN and infinities in keys and values that a row does not see: behind its end,
    before its window, in other documents of its block, in later tokens."""
    lens = [37, 64, 100] * 7
    s = _setup(dtype, lens, q, 16, 8, 64, 16, 9)
    query, kc, vc, bt, _, ks, vs = s
    starts = _starts(lens, q, 10)
    for b, n in enumerate(lens):
        first = int(starts[b].min())
        for pos in (0, first - 1, first - 2, n + q - 1):
            blk = int(bt[b, pos // 16])
            for i, c in enumerate((kc, vc)):
                if dtype == FP8:
                    c.view(torch.uint8)[blk, :, pos % 16, 3] = 0x7f
                else:
                    c[blk, :, pos % 16, 3] = float("nan") if (b + i) % 2 else float("inf")
        end = n + q
        if end % 16:
            for c in (kc, vc):
                (c.view(torch.uint8) if dtype == FP8 else c)[int(bt[b, end // 16]), :, end % 16:] = 0x7f if dtype == FP8 else float("nan")
    out = _run(s, ScoreModifiers(key_starts=starts))
    assert bool(torch.isnan(out[:, :, q - 1]).any())  # the last token sees its own
    if q > 1:
        assert not bool(torch.isnan(out[:, :, : q - 1]).any())


@pytest.mark.parametrize("dtype", [BF, HF, FP, FP8])
@pytest.mark.parametrize("bs", [8, 16, 64])
@pytest.mark.parametrize("q", [1, 40])
def test_blocks_before_a_window_are_not_read(dtype, bs, q):
    """Their table entries may be anything: no error, no effect."""
    lens = [200, 300, 77] * 7
    s = _setup(dtype, lens, q, 16, 8, 64, bs, 10)
    bt = s[3]
    for b, n in enumerate(lens):
        first = max(0, n - 50 + 1)
        bt[b, : first // bs] = torch.tensor([-7, 2**31 - 1, 10**6], dtype=torch.int32)[b % 3]
    _run(s, ScoreModifiers(window=50))
    assert read_device_errors() == 0


def test_the_lowest_values_of_the_type():
    """Keys and values at the type's ends that are seen: finite results stay finite."""
    s = _setup(BF, [40, 40], 1, 8, 2, 64, 16, 11)
    query, kc, vc, bt = s[:4]
    kc[int(bt[0, 0]), :, 3] = torch.finfo(BF).min
    vc[int(bt[1, 0]), :, 3] = torch.finfo(BF).max / 64
    _run(s, ScoreModifiers(softcap=50.0))


def test_capped_infinite_scores():
    s = _setup(BF, [40], 1, 8, 2, 64, 16, 12)
    query, kc, _, bt = s[:4]
    kc[int(bt[0, 0]), :, 3, 0] = float("inf")
    query[..., 0] = query[..., 0].abs() + 1
    out = _run(s, ScoreModifiers(softcap=10.0))
    assert bool(torch.isfinite(out).all())


def test_modifiers_rewritten_between_replays():
    """A captured step reads windows of the moment: starts and prefixes in place."""
    B, Hq, Hkv, D, bs = 2, 8, 2, 64, 16
    query, kc, vc, bt, lens, _, _ = _setup(BF, [60, 90], 1, Hq, Hkv, D, bs, 13)
    mods = ScoreModifiers(softcap=20.0, key_starts=_i32([0, 0]), prefix_lens=_i32([0, 0]))
    graph = DecodeStepGraph([kc], [vc], batch=B, max_blocks=bt.shape[1], num_q_heads=Hq, scale=D**-0.5,
                            score_modifiers=mods)
    for starts in ([0, 0], [30, 89], [59, 10]):
        mods.key_starts.copy_(_i32(starts))
        k = torch.randn(B, Hkv, 1, D).to(BF).cuda()
        slots = torch.gather(bt.long(), 1, lens.long()[:, None] // bs)[:, 0] * bs + lens % bs
        got = graph.step(block_tables=bt.cuda(), context_lens=lens.cuda(), slot_mapping=slots.cuda(), queries=[query],
                         new_keys=[k], new_values=[k])[0]
        ref, bar = attend64(query, kc, vc, bt, lens, D**-0.5, softcap=20.0, key_starts=mods.key_starts,
                            prefix_lens=mods.prefix_lens)
        check(got, ref, bar)


def test_batches_beyond_the_shared_memory_tables():
    g = torch.Generator().manual_seed(14)
    B = 9001
    kc = torch.randn(40, 1, 16, 64, generator=g).to(BF).cuda()
    bt = torch.randint(0, 40, (B, 2), generator=g).int()
    lens = torch.randint(0, 30, (B,), generator=g).int()
    q = torch.randn(B, 2, 1, 64, generator=g).to(BF).cuda()
    starts = torch.randint(0, 31, (B,), generator=g).int().cuda()
    out = paged_attention_decode(q, kc, kc, bt.cuda(), lens.cuda(), 0.125,
                                 score_modifiers=ScoreModifiers(key_starts=starts), validate=True)
    rows = [0, 2250, 4499, 4500, 9000]
    ref, bar = attend64(q[rows], kc, kc, bt[rows], lens[rows], 0.125, key_starts=starts[rows])
    check(out[rows], ref, bar)


def test_strided_inputs_and_another_stream():
    query, kc, vc, bt, lens, _, _ = _setup(BF, [40, 70], 3, 8, 2, 64, 16, 15)
    wide = torch.zeros(2, 3, 8, 130, dtype=BF, device="cuda")  # [B, q, Hq, D'], 4-byte aligned rows
    view = wide[..., 2:66].transpose(1, 2)
    view.copy_(query)
    out = torch.zeros(2, 3, 8, 66, dtype=BF, device="cuda")
    starts = torch.zeros(2, 6, dtype=torch.int32, device="cuda")
    starts[:, ::2] = _starts([40, 70], 3, 16)
    mods = ScoreModifiers(key_starts=starts[:, ::2], alibi_slopes=_slopes(8))
    bt_d, lens_d = bt.cuda(), lens.cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ws = torch.zeros(1 << 24, dtype=torch.uint8, device="cuda")
        paged_attention_decode(view, kc, vc, bt_d, lens_d, 0.125, out=out[..., :64].transpose(1, 2), workspace=ws,
                               score_modifiers=mods)
    side.synchronize()
    ref, bar = attend64(query, kc, vc, bt, lens, 0.125, key_starts=mods.key_starts, alibi_slopes=mods.alibi_slopes)
    check(out[..., :64].transpose(1, 2), ref, bar)
    assert bool((out[..., 64:] == 0).all())


def test_refusals():
    query, kc, vc, bt, lens, _, _ = _setup(BF, [40, 70], 1, 8, 2, 64, 16, 16)

    def call(mods, **kw):
        paged_attention_decode(query, kc, vc, bt.cuda(), lens.cuda(), 0.125, score_modifiers=mods, **kw)

    for mods, word in ((ScoreModifiers(softcap=-2.0), "softcap"), (ScoreModifiers(window=-2), "window"),
                       (ScoreModifiers(alibi_slopes=_slopes(4)), "alibi_slopes"),
                       (ScoreModifiers(alibi_slopes=_slopes(8).cpu()), "alibi_slopes"),
                       (ScoreModifiers(key_starts=_i32([1, 2, 3])), "key_starts"),
                       (ScoreModifiers(prefix_lens=_i32([1]).long()), "prefix_lens")):
        with pytest.raises(ValueError, match=word):
            call(mods)
    groups = PrefixGroups.from_members([[0, 1]], [16], 2, "cuda")
    with pytest.raises(ValueError, match="neither"):
        call(ScoreModifiers(window=3), prefix_groups=groups)
