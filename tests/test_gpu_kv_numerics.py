"""GPU tests of where attention's arithmetic could go wrong, against the 64-bit oracle with scores that fp32 holds exactly:
scores of any size, and of minus infinity."""
import math

import pytest
import torch

import kv_oracle as O
import nsffn as N
from test_gpu_kv_attention import E4M3, F16, Setup, assert_within, ctx, tiles  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu


def exact_scores(s, q, scale, half_out, one_p):
    """(out, bound) where every score q.k is exact in fp32 and a row's scores are equal or far apart, so that no error of
    the scores counts: P's rounding, fp32 sums of kv terms, the output's rounding."""
    out, bound = torch.zeros(s.T, s.qh, s.D, dtype=torch.float64), torch.zeros(s.T, s.qh, s.D, dtype=torch.float64)
    t = 0
    for i, (n, kv) in enumerate(s.lengths):
        k = O.sequence(s.k, s.table[i], s.page, kv, s.ks, False).repeat_interleave(s.qh // s.kh, 0)
        v = O.sequence(s.v, s.table[i], s.page, kv, s.vs, True).repeat_interleave(s.qh // s.kh, 0)
        x = q[t:t + n].double().transpose(0, 1) @ k.transpose(1, 2) * scale
        x = x.masked_fill(torch.arange(kv)[None] > torch.arange(kv - n, kv)[:, None], -math.inf)
        p = torch.softmax(x, -1)
        o = p @ v
        b = ((kv + 64) * O.U32 + 2.0 ** -20 + (O.U16 if one_p else 0.0)) * (p @ v.abs())
        b = b + (O.U16 * o.abs() + 2.0 ** -24 if half_out else 2 * O.U32 * o.abs())
        out[t:t + n], bound[t:t + n] = o.transpose(0, 1), b.transpose(0, 1)
        t += n
    return out, bound


def attend(ctx, s, q, scale, half_out, prefix=None):
    out = torch.full((s.rows, s.qh, s.D), 7.0, dtype=F16 if half_out else torch.float32, device="cuda")
    if prefix is None:
        ctx.paged_attention(s.cache, s.batch, q.cuda(), s.qh, scale, out, half_out=half_out)
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
