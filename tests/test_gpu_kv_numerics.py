"""GPU tests of where attention's arithmetic could go wrong, against the 64-bit oracle with scores that fp32 holds exactly:
scores of any size, scores of minus infinity, weights far below a row's largest, and the few-row kernel's long parts."""
import math

import pytest
import torch

import kv_oracle as O
import nsffn as N
from test_gpu_kv_attention import E4M3, F16, Setup, assert_within, ctx, tiles  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu


def exact_scores(s, q, scale, half_out, one_p, window=0):
    """(out, bound) where every score q.k is exact in fp32 and a row's scores are equal or far apart, so that no error of
    the scores counts: P's rounding, fp32 sums of kv terms, the output's rounding."""
    out, bound = torch.zeros(s.T, s.qh, s.D, dtype=torch.float64), torch.zeros(s.T, s.qh, s.D, dtype=torch.float64)
    t = 0
    for b, (n, kv) in enumerate(s.lengths):
        k = O.sequence(s.k, s.table[b], s.page, kv, s.ks, False).repeat_interleave(s.qh // s.kh, 0)
        v = O.sequence(s.v, s.table[b], s.page, kv, s.vs, True).repeat_interleave(s.qh // s.kh, 0)
        x = q[t:t + n].double().transpose(0, 1) @ k.transpose(1, 2) * scale
        i, j = torch.arange(kv - n, kv)[:, None], torch.arange(kv)[None]
        x = x.masked_fill((j > i) | (j <= i - (window or kv)), -math.inf)
        p = torch.softmax(x, -1)
        o = p @ v
        err = ((kv + 64) * O.U32 + 2.0 ** -20 + (O.U16 if one_p else 0.0)) * (p @ v.abs())
        err = err + (O.U16 * o.abs() + 2.0 ** -24 if half_out else 2 * O.U32 * o.abs())
        out[t:t + n], bound[t:t + n] = o.transpose(0, 1), err.transpose(0, 1)
        t += n
    return out, bound


def attend(ctx, s, q, scale, half_out, prefix=None, window=0):
    out = torch.full((s.rows, s.qh, s.D), 7.0, dtype=F16 if half_out else torch.float32, device="cuda")
    if prefix is None:
        ctx.paged_attention(s.cache, s.batch, q.cuda(), s.qh, scale, out, window=window, half_out=half_out)
    else:
        ctx.shared_prefix_attention(s.cache, s.batch, prefix, q.cuda(), s.qh, scale, out, half_out=half_out)
    torch.cuda.synchronize()
    return out[:s.T]


LARGE = [  # dtype, D, q heads, kv heads, page, lengths, prefix pages
    (F16, 256, 16, 8, 64, [(1, 1)], None),
    (F16, 128, 8, 4, 16, [(1, 1), (1, 3), (3, 700), (1, 2000)], None),
    (E4M3, 64, 8, 2, 64, [(4, 4), (1, 900), (2, 65)], None),
    (E4M3, 256, 4, 2, 32, [(1, 300)], None),
    (F16, 128, 8, 4, 32, [(40, 40), (33, 300), (1, 70)], None),
    (E4M3, 128, 8, 4, 64, [(64, 200), (20, 20)], None),
    (F16, 256, 8, 2, 64, [(50, 400)], None),
    (F16, 64, 4, 4, 16, [(1, 81), (1, 90), (2, 200)], 5),
    (E4M3, 128, 16, 2, 64, [(1, 200), (1, 129)], 2),
    (F16, 256, 8, 2, 16, [(30, 100), (2, 50), (1, 49)], 3),
]


@pytest.mark.parametrize("half_out", [True, False], ids=["f16", "f32"])
@pytest.mark.parametrize("top", [30.0, 1e3, 1e5, 3e6, 6e7, 1.3e8, 1e9, 1e12, 1e35, 1e39], ids=lambda x: "%.0e" % x)
@pytest.mark.parametrize("case", range(len(LARGE)))
def test_scores_of_any_size(ctx, tiles, case, top, half_out):
    """Scaled scores up to `top`, of both signs: a row's largest ones weigh alike, whatever their size, and what lies far
    below them weighs nothing.  (1e39 is beyond fp32: only the scores' differences count.)"""
    dtype, D, qh, kh, page, lengths, prefix = LARGE[case]
    s = Setup(dtype, D, qh, kh, page, lengths, seed=200 + case, shared=prefix or 0)
    # a key is 1, 1/2 or -1 times a power of two in one dim, a query an integer of 11 bits times one
    level = torch.tensor([256.0, 128.0, -256.0])
    k = torch.zeros(s.k.shape)
    k[:, :, 0, :, 0] = level[torch.randint(0, 3, k[:, :, 0, :, 0].shape, generator=s.gen)]
    s.k = k.to(dtype)
    s.device()
    q = torch.zeros(s.rows, qh, D)
    a = torch.randint(1024, 2048, (s.rows, qh), generator=s.gen)
    q[..., 0] = torch.where(torch.rand(s.rows, qh, generator=s.gen) < 0.5, a, -a).float()
    q = q.half()
    scale = top / (2047 * 256 * s.ks)
    if not scale * s.ks < 1e30:
        scale = 0.9e30 / s.ks  # the largest allowed: products of the scores reach 5e35
        q[..., 0] *= 16
        s.k = (k * (128 if dtype == F16 else 1)).to(dtype)
        s.device()
    # 30: the levels lie 15 and more apart, but the smaller queries' errors of the scores count a little
    slack = 2 * 40 * 1.45 * O.U32
    for mid, parts in ((-1, 0), (0, 1), (0, 3), (1, 1), (1, 3)):
        tiles(mid, parts)
        got = attend(ctx, s, q, scale, half_out, prefix)
        ref, bound = exact_scores(s, q, scale, half_out, half_out)
        assert_within(got, ref, bound + slack * float(s.vs * s.v.float().abs().max()))
        if s.max_q * (qh // kh) <= 16 and prefix is None:
            break


@pytest.mark.parametrize("half_out", [True, False], ids=["f16", "f32"])
@pytest.mark.parametrize("window", [1, 33, 100])
@pytest.mark.parametrize("lengths", [[(1, 300), (4, 90), (2, 2)], [(150, 400), (40, 40), (3, 70)]], ids=["few-rows", "tiles"])
def test_large_scores_in_a_window(ctx, tiles, lengths, window, half_out):
    """The same where rows of a tile have seen nothing yet beside rows of large scores, and beside rows of scores 0."""
    s = Setup(F16, 64, 8, 2, 16, lengths, seed=225, fill=math.nan)
    k = s.k.float()
    held = torch.isfinite(k)
    k[held] = 0
    level = torch.tensor([256.0, 128.0, -256.0])[torch.randint(0, 3, k[:, :, 0, :, 0].shape, generator=s.gen)]
    k[:, :, 0, :, 0] = torch.where(held[:, :, 0, :, 0], level, k[:, :, 0, :, 0])
    s.k = k.half()
    s.device()
    q = torch.zeros(s.rows, 8, 64)
    q[..., 0] = torch.randint(1024, 2048, (s.rows, 8), generator=s.gen) * torch.randint(-1, 2, (s.rows, 8), generator=s.gen)
    q = q.half()
    for top in (1e5, 1e9):
        for mid, parts in ((-1, 0), (0, 1), (0, 4), (1, 1), (1, 4)):
            tiles(mid, parts)
            got = attend(ctx, s, q, top / (2047 * 256), half_out, window=window)
            ref, bound = exact_scores(s, q, top / (2047 * 256), half_out, half_out, window)
            assert_within(got, ref, bound)


@pytest.mark.parametrize("mid", [0, 1], ids=["128", "32"])
@pytest.mark.parametrize("prefix", [None, 20])
def test_parts_that_see_only_minus_infinity(ctx, tiles, mid, prefix):
    """Keys of minus infinity weigh nothing; a row whose first parts hold nothing else is the rest's, however low the
    rest's scores are."""
    D, page, n = 64, 16, (20 if prefix is None else 1)
    lengths = [(n, 400)] if prefix is None else [(1, 330), (1, 325)]
    s = Setup(F16, D, 4, 2, page, lengths, seed=230 + mid, shared=prefix or 0)
    k = torch.zeros(s.k.shape)
    k[:, :, 0, :, 0] = -math.inf
    seen = [(int(s.table[0, p // page]), p % page) for p in (range(300, 380) if prefix is None else range(290, 320))]
    for pg, slot in seen:
        k[pg, :, 0, slot, 0] = 0
        k[pg, :, 0, slot, 1] = -2048.0
    s.k = k.half()
    s.device()
    q = torch.zeros(s.rows, 4, D)
    q[..., 0], q[..., 1] = 1.0, 2.0  # scores -512: 2^-738 against zero
    q = q.half()
    tiles(mid, 32)
    got = attend(ctx, s, q, 0.125, True, prefix).double().cpu()
    pages, slot = torch.tensor([x[0] for x in seen]), torch.tensor([x[1] for x in seen])
    v = s.v.double()[pages, :, slot // 8, :, slot % 8]  # [keys][kv heads][D]
    ref = v.mean(0).repeat_interleave(2, 0)[None].expand(s.T, 4, D)
    assert_within(got, ref, (2 * O.U16 + 2.0 ** -14) * v.abs().mean(0).repeat_interleave(2, 0)[None] + 2.0 ** -24)


@pytest.mark.parametrize("mid", [0, 1], ids=["128", "32"])
@pytest.mark.parametrize("below", [12.0, 22.6, 23.1, 24.0])
@pytest.mark.parametrize("dtype", [F16, E4M3], ids=["f16", "e4m3"])
def test_long_flat_tail_below_one_peak(ctx, tiles, dtype, below, mid):
    """One key at score 0 and 131,071 whose weights are 2^-below of its own: with fp16 outputs and more than 16 rows P is one
    fp16, subnormal from 2^-23 on, and has to count in the row's sum as it does in the product."""
    D, page, kv = 64, 64, 131072
    s = Setup(dtype, D, 4, 1, page, [(5, kv)], seed=240)
    k = torch.zeros(s.k.shape)
    k[:, :, 0, :, 0] = -16.0
    pg, slot = int(s.table[0, 0]), 5
    k[pg, :, 0, slot, 0] = 0.0
    s.k = k.to(dtype)
    q = torch.zeros(s.rows, 4, D)
    q[..., 0] = 1.0
    q = q.half()
    scale = below * math.log(2) / (16.0 * s.ks)
    tiles(mid, 1)
    sums = kv * O.U32  # a lane adds half the row's keys two at a time, a step off by a unit at most, the product 16 at a time
    # all values equal: whatever the weights are, their sum has to be the products'
    v = torch.ones(s.v.shape) / s.vs
    s.v = v.to(dtype)
    s.device()
    got = attend(ctx, s, q, scale, True).double().cpu()
    assert_within(got, torch.ones_like(got), torch.full_like(got, sums + 2.0 ** -20 + O.U16 + 2.0 ** -24))
    # the peak's value zero: the tail's share, P within half a step of fp16 (2^-25 of its subnormals; the peak is 2^9)
    v[pg, :, slot // O.CHUNK[dtype], :, slot % O.CHUNK[dtype]] = 0
    s.v = v.to(dtype)
    s.device()
    got = attend(ctx, s, q, scale, True).double().cpu()
    tail = (kv - torch.arange(5, 0, -1)).double() * 2.0 ** -below  # keys that row i sees but the peak
    ref = (tail / (1 + tail))[:, None, None].expand(5, 4, D)
    half_step = max(O.U16, 2.0 ** -25 / 2.0 ** (9.0 - below))
    assert_within(got, ref, ref * (2 * sums + 2.0 ** -20 + 2 * half_step + O.U16 + 8 * O.U32 * below) + 2.0 ** -25)


LONG = [  # dtype, D, q heads, kv heads, page, lengths, window
    (F16, 64, 8, 8, 64, [(1, 20001)], 0),
    (F16, 64, 8, 8, 16, [(1, 20000)], 0),
    (F16, 256, 16, 8, 64, [(1, 12345)], 0),
    (F16, 128, 16, 8, 256, [(2, 15000)], 12000),
    (F16, 64, 8, 8, 16, [(1, 26000)], 25000),
    (E4M3, 64, 16, 8, 64, [(1, 40000)], 0),
    (E4M3, 64, 16, 8, 16, [(2, 35001)], 0),
    (E4M3, 128, 8, 8, 32, [(1, 24000)], 20000),
    (E4M3, 256, 8, 8, 128, [(1, 20000)], 0),
    (F16, 64, 8, 8, 32, [(1, 30000), (1, 5), (2, 9000), (0, 7), (1, 300)], 0),
    (E4M3, 64, 8, 8, 64, [(1, 9000), (1, 33000)], 0),
    (F16, 256, 16, 1, 64, [(1, 6000)], 0),   # 16 rows over 47 parts: the join takes them in three rounds
    (E4M3, 256, 8, 1, 64, [(2, 11000)], 0),
]


@pytest.mark.parametrize("half_out", [True, False], ids=["f16", "f32"])
@pytest.mark.parametrize("case", range(len(LONG)))
def test_long_sequences_of_few_rows(ctx, case, half_out):
    """Parts of more than four key tiles (a wave takes several, its maximum running over them) and joins of more parts
    than a round takes, with keys of far larger scores late, in the middle or early."""
    dtype, D, qh, kh, page, lengths, window = LONG[case]
    at = (0.97, 0.5, 0.3)[(case + half_out) % 3]  # a window's start lies below all of them
    s = Setup(dtype, D, qh, kh, page, lengths, seed=260 + case)
    for i, (_, kv) in enumerate(lengths):
        p = int(at * (kv - 1))
        pg, slot = int(s.table[i, p // page]), p % page
        row = (s.k[pg, :, :, slot].float() * 4).clamp(-448 if dtype == E4M3 else -65504, 448 if dtype == E4M3 else 65504)
        O.raw(s.k)[pg, :, :, slot] = O.raw(row.to(dtype))  # one key of scores some 4 times the others'
    s.device()
    q = s.queries()
    got = s.attend(ctx, q.cuda(), window, half_out)
    torch.cuda.synchronize()
    ref, bound = O.attention(q[:s.T], s.k, s.v, s.table, s.lengths, page, D ** -0.5, window, s.ks, s.vs, half_out, one_p=False)
    assert_within(got, ref, bound)
