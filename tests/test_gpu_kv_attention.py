"""GPU tests of ns_kv_append, ns_paged_attention and ns_shared_prefix_attention through the C ABI against the 64-bit
oracle (tests/kv_oracle.py), with bounds by arithmetic: types, head layouts, pages, ragged lengths, windows, garbage
in unused slots, contradicting descriptions, graphs, streams, and the calls together as a layer runs them."""
import numpy as np
import pytest
import torch

import kv_oracle as O
import nsffn as N

pytestmark = pytest.mark.gpu

F16, E4M3 = torch.float16, torch.float8_e4m3fn
NAN = float("nan")


@pytest.fixture(scope="module")
def ctx():
    assert torch.cuda.is_available(), "GPU tests need a visible MI355X"
    c = N.Context(0)
    yield c
    torch.cuda.synchronize()
    c.close()


class Setup:
    """A cache of random values and a batch: host copies beside device tensors."""

    def __init__(self, dtype, D, qh, kh, page, lengths, seed=0, fill=None, shared=0, tokens=None, max_q=None, max_kv=None):
        gen = torch.Generator().manual_seed(seed)
        self.dtype, self.D, self.qh, self.kh, self.page, self.lengths = dtype, D, qh, kh, page, lengths
        self.ks, self.vs = (1.0, 1.0) if dtype == F16 else (0.0625, 0.03125)
        self.table, self.pages = O.page_tables(lengths, page, seed=seed, shared=shared)
        shapes = N.kv_shapes(self.pages, page, kh, D, N.KV_F16 if dtype == F16 else N.KV_E4M3)
        self.k, self.v = ((torch.randn(s, generator=gen) / x).to(dtype) for s, x in zip(shapes, (self.ks, self.vs)))
        if fill is not None:  # everything that no sequence holds
            for cache, values in ((self.k, False), (self.v, True)):
                held = [(kv, kv) for _, kv in lengths]
                keep = O.read_new(cache, self.table, held, page, values)
                O.raw(cache).fill_(fill)
                pg, slot = O.slots(self.table, held, page)
                c = O.CHUNK[dtype]
                if values:
                    O.raw(cache)[pg, :, slot // c, :, slot % c] = O.raw(keep)
                else:
                    O.raw(cache)[pg, :, :, slot] = O.raw(keep).unflatten(2, (D // c, c))
        self.starts = O.starts(lengths)
        self.T = int(self.starts[-1])
        self.rows = tokens or max(1, self.T)
        self.max_q = max_q or max(1, max(n for n, _ in lengths))
        self.max_kv = max_kv or max(1, max(kv for _, kv in lengths))
        self.gen = gen
        self.device()

    def device(self):
        self.dk, self.dv = self.k.cuda(), self.v.cuda()
        self.dtable, self.dstarts = self.table.cuda(), self.starts.cuda()
        self.dlen = torch.tensor([kv for _, kv in self.lengths], dtype=torch.int32).cuda()
        self.cache = N.KvCache(self.dk, self.dv, self.page, self.kh, self.D, self.ks, self.vs)
        self.batch = N.KvBatch(self.dtable, self.dstarts, self.dlen, self.rows, self.max_q, self.max_kv)

    def queries(self, spread=1.5):
        return (torch.randn(self.rows, self.qh, self.D, generator=self.gen) * spread).half()

    def attend(self, ctx, q, window=0, half_out=True, prefix=None, out=None, stream=None):
        if out is None:
            out = torch.full((self.rows, self.qh, self.D), 7.0, dtype=torch.float16 if half_out else torch.float32, device="cuda")
        scale = self.D ** -0.5
        if prefix is None:
            ctx.paged_attention(self.cache, self.batch, q, self.qh, scale, out, window=window, half_out=half_out, stream=stream)
        else:
            ctx.shared_prefix_attention(self.cache, self.batch, prefix, q, self.qh, scale, out, half_out=half_out, stream=stream)
        return out

    def expect(self, q, window=0, half_out=True):
        # rows of a sequence and key head above 16 take P as one fp16 where the output is one
        return O.attention(q[:self.T], self.k, self.v, self.table, self.lengths, self.page, self.D ** -0.5, window, self.ks,
                           self.vs, half_out, one_p=half_out)


def assert_within(got, ref, bound):
    got = got.double().cpu()
    bad = ~((got - ref).abs() <= bound)
    if bad.any():
        i = tuple(int(x) for x in bad.nonzero()[0])
        raise AssertionError(f"{int(bad.sum())} of {bad.numel()} outside, first at {i}: {float(got[i])} for {float(ref[i])}, "
                             f"bound {float(bound[i])}")


def attention_case(ctx, s, window=0, half_out=True, prefix=None):
    q = s.queries()
    out = s.attend(ctx, q.cuda(), window, half_out, prefix)
    torch.cuda.synchronize()
    ref, bound = s.expect(q, window, half_out)
    assert_within(out[:s.T], ref, bound)
    assert bool((out[s.T:] == 7.0).all()), "rows behind the last sequence"


# ---- append -----------------------------------------------------------------------------------------------

APPENDS = [  # dtype, D, q heads, kv heads, page, lengths, rot, pairs, norm
    (F16, 256, 16, 8, 64, [(1, 1)], 256, False, True),
    (F16, 256, 16, 8, 64, [(1, 2206)], 256, False, True),
    (E4M3, 128, 32, 8, 16, [(4, 100), (1, 17), (0, 5), (3, 16), (2, 33)], 64, True, False),
    (F16, 64, 9, 3, 16, [(23, 30), (8, 8), (16, 24)], 32, False, True),
    (E4M3, 256, 8, 1, 32, [(37, 37), (1, 15), (17, 200)], 256, False, True),
    (F16, 128, 5, 5, 256, [(300, 700)], 128, True, True),
    (E4M3, 64, 3, 3, 16, [(16, 16), (16, 48), (31, 47)], 8, False, False),
    (F16, 256, 2, 1, 128, [(3, 262144)], 256, False, False),
    (F16, 128, 4, 2, 16, [(1, 40 + i) for i in range(70)] + [(0, 9), (2, 2)], 0, False, True),
]


@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append(ctx, case):
    dtype, D, qh, kh, page, lengths, rot, pairs, norm = APPENDS[case]
    s = Setup(dtype, D, qh, kh, page, lengths, seed=case, tokens=O.starts(lengths)[-1].item() + 2)
    q, k, v = (torch.randn(s.rows, h, D, generator=s.gen) * x for h, x in ((qh, 1.7), (kh, 1.3), (kh, 0.8)))
    w = [1 + 0.2 * torch.randn(D, generator=s.gen) for _ in range(2)] + [torch.ones(D)] if norm else [None] * 3
    freqs = torch.from_numpy(N.rope_freqs(1e6, rot)) if rot else torch.zeros(1)
    q_out = torch.full((s.rows, qh, D), 7.0, dtype=torch.float16, device="cuda")
    dev = [None if x is None else x.cuda() for x in w]
    ctx.kv_append(s.cache, s.batch, q.cuda(), k.cuda(), v.cuda(), qh, freqs.cuda(), rot, q_out, q_norm=dev[0], k_norm=dev[1],
                  v_norm=dev[2], eps=1e-6, rope=N.ROPE_PAIRS if pairs else N.ROPE_HALVES)
    torch.cuda.synchronize()
    _, pos = O.positions(lengths)
    # fp32 on the way: the norm's sum of D squares, root and quotient, two products; the turn's fraction (2^-24 of
    # half a turn: pi 2^-24), sine and cosine (2 ulp each), two products and a sum
    chain = ((D / 2 + 8) if norm else 0) + 16
    half_step = {F16: (O.U16, 2.0 ** -25), E4M3: (O.U8, 2.0 ** -10)}[dtype]

    def check(got, u, weight, turn, scale, step):
        x, mag = O.rotated(O.normed(u[:s.T], weight, 1e-6), pos, freqs, rot if turn else 0, pairs)
        x, mag = x / scale, mag / scale
        if step[0] == O.U8:
            x = x.clamp(-O.E4M3_MAX, O.E4M3_MAX)
        err = chain * O.U32 * mag
        assert_within(got[:s.T].float(), x, err + step[0] * (x.abs() + err) + step[1])

    check(q_out, q, w[0], True, 1.0, (O.U16, 2.0 ** -25))
    assert bool((q_out[s.T:] == 7.0).all())
    k_new, v_new = s.dk.cpu(), s.dv.cpu()
    check(O.read_new(k_new, s.table, lengths, page, False), k, w[1], True, s.ks, half_step)
    check(O.read_new(v_new, s.table, lengths, page, True), v, w[2], False, s.vs, half_step)
    for new, old, values in ((k_new, s.k, False), (v_new, s.v, True)):  # every other slot keeps its bits
        assert torch.equal(O.without_new(new, s.table, lengths, page, values), O.without_new(old, s.table, lengths, page, values))


@pytest.mark.parametrize("dtype", [F16, E4M3])
def test_append_rounds_to_nearest(ctx, dtype):
    """Without norm and rotation the stored values are the roundings of the inputs: ties, subnormals, the largest
    values, saturation (e4m3) and overflow (fp16), infinities and NaN, for one token and for whole groups."""
    D, heads, page, lengths = 256, 2, 16, [(16, 16), (1, 6)]
    s = Setup(dtype, D, 2, heads, page, lengths, seed=5)
    s.ks = s.vs = 1.0
    s.device()
    if dtype == E4M3:
        grid = torch.arange(256, dtype=torch.uint8).view(E4M3).float()
        grid = grid[torch.isfinite(grid)].unique()
    else:
        grid = torch.randint(0, 0x7C00, (4000,), generator=s.gen, dtype=torch.int32).short().view(torch.float16).float().unique()
    mid = (grid[1:] + grid[:-1]) / 2
    vals = torch.cat([grid, mid, torch.nextafter(mid, mid + 1), torch.nextafter(mid, mid - 1), -mid,
                      torch.tensor([0.0, -0.0, 447.9, 448.0, 449.0, 463.9, 464.0, 465.0, 1e4, -1e9, 65504.0, 65519.9, 65520.0, NAN,
                                    float("inf"), -float("inf"), 2.0 ** -10, 2.0 ** -11, 3.1e-8])])
    n = s.rows * heads * D
    u = vals[torch.randint(0, len(vals), (n,), generator=s.gen)].view(s.rows, heads, D)
    u.view(-1)[:len(vals)] = vals[:n]
    q_out = torch.empty(s.rows, 2, D, dtype=torch.float16, device="cuda")
    ctx.kv_append(s.cache, s.batch, u.cuda(), u.cuda(), u.cuda(), 2, None, 0, q_out)
    torch.cuda.synchronize()
    assert torch.equal(q_out.cpu().nan_to_num(nan=1.25), u.half().nan_to_num(nan=1.25))
    ref = torch.where(u.isnan(), u, u.clamp(-O.E4M3_MAX, O.E4M3_MAX)).to(E4M3) if dtype == E4M3 else u.half()
    for cache, values in ((s.dk, False), (s.dv, True)):
        got = O.read_new(cache.cpu(), s.table, lengths, page, values)
        assert torch.equal(got.float().nan_to_num(nan=1.25, posinf=9e9, neginf=-9e9), ref.float().nan_to_num(nan=1.25, posinf=9e9, neginf=-9e9))


def test_append_keys_and_values_only(ctx):
    lengths = [(5, 21), (1, 3)]
    a, b = (Setup(F16, 128, 8, 4, 16, lengths, seed=6) for _ in range(2))
    q, k, v = (torch.randn(a.rows, h, 128, generator=a.gen).cuda() for h in (8, 4, 4))
    freqs = torch.from_numpy(N.rope_freqs(1e4, 128)).cuda()
    q_out = torch.empty(a.rows, 8, 128, dtype=torch.float16, device="cuda")
    ctx.kv_append(a.cache, a.batch, q, k, v, 8, freqs, 128, q_out)
    ctx.kv_append(b.cache, b.batch, None, k, v, 8, freqs, 128, None)
    torch.cuda.synchronize()
    assert torch.equal(a.dk, b.dk) and torch.equal(a.dv, b.dv) and not torch.equal(a.dk.cpu(), a.k)


def test_append_contradicting_sequences_and_pages(ctx):
    """Sequences whose description does not hold get NaN queries and store nothing; a page outside the cache is not
    written; the sequences beside them are as they would be alone."""
    lengths = [(2, 20), (3, 40), (2, 18), (1, 33), (2, 17)]
    s = Setup(F16, 64, 4, 2, 16, lengths, seed=7, max_q=2, max_kv=40)
    s.dlen[2] = 41                      # above max_kv
    s.dlen[4] = 1                       # fewer than the new tokens
    s.dtable[3, 2] = s.pages            # position 32 of sequence 3
    q, k, v = (torch.randn(s.rows, h, 64, generator=s.gen) for h in (4, 2, 2))
    q_out = torch.full((s.rows, 4, 64), 7.0, dtype=torch.float16, device="cuda")
    ctx.kv_append(s.cache, s.batch, q.cuda(), k.cuda(), v.cuda(), 4, None, 0, q_out)
    torch.cuda.synchronize()
    got = q_out.cpu()
    rows = torch.tensor([0, 0, 1, 1, 1, 2, 2, 3, 4, 4])
    nan = (rows == 1) | (rows == 2) | (rows == 4)  # sequence 1 has more than max_q new tokens
    assert got[nan].isnan().all() and torch.equal(got[~nan], q.half()[~nan])
    only = [(2, 20)]
    ref = s.k.clone()
    pg, slot = O.slots(s.table, only, 16)
    ref[pg, :, :, slot] = k[:2].half().view(2, 2, 8, 8)
    assert torch.equal(s.dk.cpu(), ref)


# ---- attention --------------------------------------------------------------------------------------------

ATTENTION = [  # dtype, D, q heads, kv heads, page, lengths, window
    (F16, 256, 16, 8, 64, [(1, 1)], 0),
    (F16, 256, 16, 8, 64, [(1, 2206)], 0),
    (F16, 256, 16, 8, 16, [(1, 31), (1, 32), (1, 33), (1, 64), (1, 65), (0, 40), (1, 129), (1, 500)], 0),
    (E4M3, 256, 16, 8, 16, [(1, 15), (1, 16), (1, 17), (1, 63), (1, 64), (1, 65), (3, 300)], 0),
    (F16, 128, 32, 8, 32, [(4, 100), (1, 999), (2, 2), (3, 258)], 0),
    (E4M3, 128, 32, 8, 128, [(4, 1000), (1, 130), (2, 2)], 100),
    (F16, 64, 12, 12, 16, [(16, 16), (1, 1), (7, 200)], 0),
    (E4M3, 64, 9, 3, 256, [(5, 5), (1, 700), (2, 300)], 33),
    (F16, 256, 16, 1, 64, [(1, 333), (1, 1)], 0),
    (F16, 128, 28, 4, 64, [(2, 444), (1, 70)], 1),
    (F16, 256, 16, 8, 64, [(157, 405)], 0),
    (F16, 256, 16, 8, 16, [(64, 64), (65, 65), (1, 200), (100, 333), (0, 0), (9, 40)], 0),
    (E4M3, 256, 4, 2, 32, [(200, 300), (33, 33)], 0),
    (F16, 128, 8, 2, 32, [(129, 129), (31, 500)], 50),
    (E4M3, 128, 40, 8, 16, [(77, 80), (1, 300), (13, 13)], 64),
    (F16, 64, 3, 3, 16, [(40, 41), (17, 2000)], 0),
    (E4M3, 64, 8, 1, 64, [(50, 90), (2, 150), (300, 301)], 70),
    (F16, 64, 32, 1, 16, [(1, 90), (2, 50)], 0),      # 32 heads a group: a single token is many rows
    (F16, 128, 16, 8, 16, [(1, 20 + 3 * i) for i in range(70)] + [(0, 0)] * 60 + [(2, 600), (1, 1)], 0),
]


@pytest.mark.parametrize("half_out", [True, False], ids=["f16", "f32"])
@pytest.mark.parametrize("case", range(len(ATTENTION)))
def test_attention(ctx, case, half_out):
    dtype, D, qh, kh, page, lengths, window = ATTENTION[case]
    s = Setup(dtype, D, qh, kh, page, lengths, seed=20 + case, tokens=O.starts(lengths)[-1].item() + 3)
    attention_case(ctx, s, window, half_out)


@pytest.fixture
def tiles(ctx):
    """tiles(mid, parts): the row tiles' kernel and their key parts for this test."""
    def set_(mid, parts):
        ctx.set_tuning("attn_mid", mid)
        ctx.set_tuning("attn_parts", parts)
    yield set_
    set_(-1, 0)


@pytest.mark.parametrize("half_out", [True, False], ids=["f16", "f32"])
@pytest.mark.parametrize("mid,parts", [(0, 1), (0, 3), (0, 32), (1, 1), (1, 2), (1, 7)])
@pytest.mark.parametrize("case", [10, 11, 12, 13, 14, 15, 16, 17])
def test_row_tiles(ctx, tiles, case, mid, parts, half_out):
    """Both kernels for many rows, whichever is planned, with one key part, few and more than there are tiles; unused
    slots are NaN."""
    dtype, D, qh, kh, page, lengths, window = ATTENTION[case]
    s = Setup(dtype, D, qh, kh, page, lengths, seed=150 + case, fill=NAN if dtype == F16 else 0x7F)
    tiles(mid, parts)
    attention_case(ctx, s, window, half_out)


@pytest.mark.parametrize("mid,parts", [(0, 1), (0, 5), (1, 1), (1, 6)])
@pytest.mark.parametrize("case", [0, 2, 4, 5])
def test_shared_prefix_row_tiles(ctx, tiles, case, mid, parts):
    dtype, D, qh, kh, page, prefix, own = SHARED[case]
    lengths = [(n, prefix * page + kv) for n, kv in own]
    s = Setup(dtype, D, qh, kh, page, lengths, seed=170 + case, fill=NAN if dtype == F16 else 0x7F, shared=prefix)
    tiles(mid, parts)
    attention_case(ctx, s, 0, True, prefix)


@pytest.mark.parametrize("half_out", [True, False], ids=["f16", "f32"])
@pytest.mark.parametrize("case", [2, 3, 5, 7, 11, 12, 13, 16])
def test_slots_outside_the_sequences_may_hold_anything(ctx, case, half_out):
    """Every byte that no sequence holds is NaN (0xFF / 0x7F bytes are NaN in both types), and table entries of pages
    wholly before every row's window are outside the cache."""
    dtype, D, qh, kh, page, lengths, window = ATTENTION[case]
    s = Setup(dtype, D, qh, kh, page, lengths, seed=40 + case, fill=NAN if dtype == F16 else 0x7F)
    if window:
        for i, (n, kv) in enumerate(lengths):
            dead = max(0, kv - n - window + 1) // page
            s.dtable[i, :dead] = 1 << 30
    attention_case(ctx, s, window, half_out)


def test_bounds_above_the_lengths(ctx):
    """max_q and max_kv are bounds: results with generous ones are within the same error."""
    lengths = [(1, 300), (20, 50), (2, 2)]
    s = Setup(F16, 128, 16, 4, 16, lengths, seed=60, max_q=20, max_kv=300)
    s.dtable = torch.cat([s.dtable, torch.full((3, 100), -1, dtype=torch.int32, device="cuda")], 1).contiguous()
    s.batch = N.KvBatch(s.dtable, s.dstarts, s.dlen, s.rows, 2000, 1900)
    attention_case(ctx, s)


def test_windows_as_long_as_the_context(ctx):
    """Windows that hold every position, up to the largest number, are no window."""
    s = Setup(F16, 128, 8, 4, 16, [(1, 300), (40, 120)], seed=66)
    q = s.queries().cuda()
    whole = s.attend(ctx, q).clone()
    for window in (300, 301, 1 << 31, (1 << 32) - 1):
        assert torch.equal(s.attend(ctx, q, window=window), whole)
    with pytest.raises(ValueError, match="window"):
        s.attend(ctx, q, window=-1)


def test_binding_refuses_short_tensors(ctx):
    s = Setup(F16, 64, 4, 2, 16, [(3, 20)], seed=67)
    q = s.queries().cuda()
    with pytest.raises(ValueError, match="smaller"):
        s.attend(ctx, q[:2])
    with pytest.raises(ValueError, match="smaller"):
        s.attend(ctx, q, out=torch.empty(2, 4, 64, dtype=torch.float16, device="cuda"))
    with pytest.raises(TypeError):
        N.KvCache(s.dk.transpose(0, 1), s.dv, 16, 2, 64)
    with pytest.raises(ValueError, match="whole pages"):
        N.KvCache(s.dk, s.dv, 16, 3, 64)
    with pytest.raises(ValueError, match="do not match"):
        N.KvBatch(s.dtable, s.dstarts[:1], s.dlen, 3, 3, 20)


def test_binding_refuses_values_of_another_type(ctx):
    """fp32 queries (what ns_qkv leaves), an output of the other type, fp64 frequencies and bf16 are refused by the calls."""
    s = Setup(F16, 64, 4, 2, 16, [(3, 20)], seed=68)
    q = s.queries().cuda()
    for bad in (q.float(), q.bfloat16()):
        with pytest.raises(TypeError, match="float16"):
            s.attend(ctx, bad)
        with pytest.raises(TypeError, match="float16"):
            s.attend(ctx, bad, prefix=0)
    with pytest.raises(TypeError, match="float16"):
        s.attend(ctx, q, out=torch.empty(3, 4, 64, device="cuda"))
    with pytest.raises(TypeError, match="float32"):
        s.attend(ctx, q, half_out=False, out=torch.empty(6, 4, 64, dtype=F16, device="cuda"))
    x = [torch.randn(3, h, 64, device="cuda") for h in (4, 2, 2)]
    freqs, before = torch.ones(32, device="cuda"), s.dk.clone()
    for i, bad in ((0, x[0].double()), (1, torch.zeros(12, 2, 64, dtype=F16, device="cuda"))):
        with pytest.raises(TypeError, match="float32"):
            ctx.kv_append(s.cache, s.batch, *x[:i], bad, *x[i + 1:], 4, freqs, 64, q)
    with pytest.raises(TypeError, match="float32"):
        ctx.kv_append(s.cache, s.batch, *x, 4, freqs.double(), 64, q)
    with pytest.raises(TypeError, match="float16"):
        ctx.kv_append(s.cache, s.batch, *x, 4, freqs, 64, q.float())
    assert torch.equal(s.dk, before)


@pytest.mark.parametrize("many", [False, True], ids=["few-rows", "tiles"])
def test_contradicting_sequences_and_pages_are_nan(ctx, many):
    n = 20 if many else 2
    lengths = [(n, 50), (n, 60), (n, 70), (n, 80), (n, 40)]
    s = Setup(F16, 128, 4, 2, 16, lengths, seed=61)
    q = s.queries()
    ref, bound = s.expect(q)
    s.dlen[1] = n - 1                     # fewer than its new tokens
    s.dlen[2] = s.max_kv + 1              # above the bound
    s.dtable[3, 1] = -5                   # a page that all its rows see
    s.dtable[3, 2] = s.pages
    out = s.attend(ctx, q.cuda())
    torch.cuda.synchronize()
    good = torch.zeros(s.T, dtype=torch.bool)
    good[:n] = good[4 * n:] = True
    assert_within(out.cpu()[good], ref[good], bound[good])
    assert out.cpu()[~good].isnan().all()


@pytest.mark.parametrize("prefix", [None, 1])
def test_more_new_tokens_than_the_bound(ctx, prefix):
    """A sequence with more new tokens than max_q is NaN whichever kernel its rows would have gone to; the others are
    as they should be."""
    lengths = [(1, 20), (30, 47), (2, 22)]
    s = Setup(F16, 128, 4, 2, 16, lengths, seed=65, max_q=2, shared=prefix or 0)
    q = s.queries()
    out = s.attend(ctx, q.cuda(), prefix=prefix).cpu()
    ref, bound = s.expect(q)
    assert out[1:31].isnan().all()
    keep = [0, 31, 32]
    assert_within(out[keep], ref[keep], bound[keep])


def test_nan_and_infinite_values(ctx):
    """A key or value that a row sees acts as in the definition: NaN reaches it, and a sequence beside it is untouched."""
    lengths = [(1, 40), (1, 40)]
    s = Setup(F16, 64, 2, 2, 16, lengths, seed=62)
    pg, slot = O.slots(s.table, [(1, 20), (0, 0)], 16)
    s.dv[pg[0], 0, slot[0] // 8, 5, slot[0] % 8] = NAN
    s.dk[pg[0], 1, 0, slot[0], 3] = NAN
    q = s.queries()
    out = s.attend(ctx, q.cuda()).cpu()
    ref, bound = s.expect(q)
    assert out[0, 0, 5].isnan() and out[0, 1].isnan().all()
    keep = torch.arange(64) != 5
    assert_within(out[0, 0][keep], ref[0, 0][keep], bound[0, 0][keep])
    assert_within(out[1], ref[1], bound[1])


@pytest.mark.parametrize("half_out", [True, False], ids=["f16", "f32"])
@pytest.mark.parametrize("spread", [0.0, 12.0])
def test_flat_and_peaked_scores(ctx, spread, half_out):
    """All scores equal, and scores hundreds apart (the running maximum moves far; most weights vanish)."""
    for lengths in ([(1, 700)], [(40, 300)]):
        s = Setup(F16, 128, 8, 4, 32, lengths, seed=63)
        q = s.queries(spread)
        out = s.attend(ctx, q.cuda(), half_out=half_out)
        torch.cuda.synchronize()
        ref, bound = s.expect(q, half_out=half_out)
        assert_within(out, ref, bound)


def test_offsets_past_32_bits(ctx):
    """A cache of 5 GB a side whose sequence lies in its last pages."""
    D, kh, page = 256, 8, 256
    pages = 5000
    shapes = N.kv_shapes(pages, page, kh, D)
    assert np.prod(shapes[0]) * 2 > 1 << 32
    k, v = (torch.empty(x, dtype=F16, device="cuda") for x in shapes)
    lengths = [(3, 600), (40, 300)]
    s = Setup(F16, D, 16, kh, page, lengths, seed=64)
    s.dtable = torch.where(s.table >= 0, s.table + pages - s.pages, s.table).cuda()
    k[pages - s.pages:], v[pages - s.pages:] = s.dk, s.dv
    s.cache = N.KvCache(k, v, page, kh, D)
    s.batch = N.KvBatch(s.dtable, s.dstarts, s.dlen, s.rows, s.max_q, s.max_kv)
    q, kn, vn = (torch.randn(s.rows, h, D, generator=s.gen) for h in (16, kh, kh))
    q_out = torch.empty(s.rows, 16, D, dtype=F16, device="cuda")
    ctx.kv_append(s.cache, s.batch, q.cuda(), kn.cuda(), vn.cuda(), 16, None, 0, q_out)
    torch.cuda.synchronize()
    s.k, s.v = k[pages - s.pages:].cpu(), v[pages - s.pages:].cpu()
    assert torch.equal(O.read_new(s.k, s.table, lengths, page, False), kn.half())
    assert torch.equal(O.read_new(s.v, s.table, lengths, page, True), vn.half())
    attention_case(ctx, s)


# ---- shared prefix ----------------------------------------------------------------------------------------

SHARED = [  # dtype, D, q heads, kv heads, page, prefix pages, lengths behind the prefix
    (F16, 256, 16, 8, 64, 4, [(1, 10), (1, 1), (1, 77)]),
    (F16, 256, 16, 8, 16, 1, [(1, 1), (1, 16), (0, 4), (1, 17)]),
    (E4M3, 256, 16, 2, 16, 9, [(2, 20), (1, 300), (4, 4)]),
    (F16, 128, 32, 8, 32, 20, [(1, 5 + 7 * i) for i in range(40)]),
    (E4M3, 128, 28, 4, 64, 3, [(9, 100), (1, 1), (30, 30)]),
    (F16, 64, 12, 12, 16, 33, [(17, 17), (1, 60), (40, 41)]),
    (E4M3, 64, 8, 1, 128, 5, [(1, 3)] * 80 + [(3, 200)]),
    (F16, 128, 8, 4, 16, 7, [(1, 100)]),
]


@pytest.mark.parametrize("half_out", [True, False], ids=["f16", "f32"])
@pytest.mark.parametrize("case", range(len(SHARED)))
def test_shared_prefix(ctx, case, half_out):
    dtype, D, qh, kh, page, prefix, own = SHARED[case]
    lengths = [(n, prefix * page + kv) for n, kv in own]
    s = Setup(dtype, D, qh, kh, page, lengths, seed=80 + case, fill=NAN if dtype == F16 else 0x7F, shared=prefix,
              tokens=O.starts(lengths)[-1].item() + 2)
    attention_case(ctx, s, 0, half_out, prefix)
    attention_case(ctx, s, 0, half_out, 0)  # no shared pages: the plain call


def test_shared_prefix_contradictions(ctx):
    """A sequence that ends inside the prefix gets NaN rows, a bad page in the prefix makes all rows NaN."""
    lengths = [(1, 80), (1, 70), (2, 90)]
    s = Setup(F16, 128, 8, 4, 16, lengths, seed=95, shared=4)
    q = s.queries()
    ref, bound = s.expect(q)
    s.dlen[1] = 64
    out = s.attend(ctx, q.cuda(), prefix=4).cpu()
    assert out[1].isnan().all()
    assert_within(out[[0, 2, 3]], ref[[0, 2, 3]], bound[[0, 2, 3]])
    s.dtable[0, 1] = -1
    assert s.attend(ctx, q.cuda(), prefix=4).isnan().all()


def drawn_call(seed):
    """A call of random sizes: type, heads, pages, a ragged batch, window or prefix, bounds above the lengths."""
    r = np.random.RandomState(seed)
    pick = lambda *x: x[r.randint(len(x))]
    dtype, D, page = pick(F16, E4M3), int(pick(64, 128, 256)), int(pick(16, 32, 64, 256))
    kh, group = int(pick(1, 2, 3, 8)), int(pick(1, 2, 3, 4, 7, 16))
    prefix = int(pick(0, 0, 0, 1, 5, 20))
    lengths = []
    for _ in range(pick(1, 1, 2, 5, 12, 70)):
        n = int(pick(0, 1, 1, 2, r.randint(1, 20), r.randint(1, 300)))
        lengths.append((n, prefix * page + n + int(pick(0, 0, 1, r.randint(1, 70), r.randint(1, 1500)))))
    if sum(n for n, _ in lengths) * group * kh > 6000:  # the oracle's time
        lengths = lengths[:5]
    lengths[0] = (max(1, lengths[0][0]), lengths[0][1] + 1)
    window = 0 if prefix else int(pick(0, 0, 1, 16, r.randint(2, 200), 1024))
    s = Setup(dtype, D, kh * group, kh, page, lengths, seed=seed, fill=NAN if dtype == F16 else 0x7F, shared=prefix,
              tokens=sum(n for n, _ in lengths) + int(pick(0, 1, 40)))
    if r.randint(2):  # bounds that the lengths stay below, as a captured step has them
        s.batch = N.KvBatch(s.dtable, s.dstarts, s.dlen, s.rows, s.max_q + int(pick(1, 30)), s.table.shape[1] * page)
    return s, window, bool(r.randint(2)), prefix or None


@pytest.mark.parametrize("seed", range(40))
def test_drawn_calls(ctx, seed):
    s, window, half_out, prefix = drawn_call(seed)
    attention_case(ctx, s, window, half_out, prefix)


# ---- together, graphs, streams ------------------------------------------------------------------------------

def test_same_inputs_give_the_same_bits(ctx):
    for lengths, prefix in (([(1, 5000)], None), ([(157, 405)], None), ([(1, 700)] * 6, 4), ([(30, 700)] * 2, 4)):
        s = Setup(F16, 256, 16, 8, 64, lengths, seed=100, shared=prefix or 0)
        q = s.queries().cuda()
        first = s.attend(ctx, q, prefix=prefix).clone()
        for _ in range(5):
            assert torch.equal(s.attend(ctx, q, prefix=prefix), first)


@pytest.mark.parametrize("shape", ["decode", "prompt", "shared"])
def test_captured_steps_follow_the_buffers(ctx, shape):
    """append and attention captured once: replays on new lengths, tables and inputs in the same buffers equal eager
    calls on them."""
    D, qh, kh, page = 128, 8, 4, 16
    prefix = 3 if shape == "shared" else None
    n = 30 if shape == "prompt" else 1
    base = 3 * page if prefix else 0
    lengths = [(n, base + 200 + n)] * 3  # pages for every length that a replay sets
    s = Setup(F16, D, qh, kh, page, lengths, seed=101, shared=prefix or 0)
    x = [torch.zeros(s.rows, h, D, device="cuda") for h in (qh, kh, kh)]
    q_out = torch.zeros(s.rows, qh, D, dtype=F16, device="cuda")
    out = torch.zeros(s.rows, qh, D, dtype=F16, device="cuda")
    freqs = torch.from_numpy(N.rope_freqs(1e4, D)).cuda()

    def step(stream=None):
        ctx.kv_append(s.cache, s.batch, *x, qh, freqs, D, q_out, stream=stream)
        s.attend(ctx, q_out, prefix=prefix, out=out, stream=stream)

    step()  # sizes the workspace
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        for t in x:
            t.copy_(torch.randn(t.shape, generator=s.gen))
        s.dlen.copy_(torch.tensor([base + n + (37 * i + 50 * j) % 190 for j in range(3)], dtype=torch.int32))
        k0, v0 = s.dk.clone(), s.dv.clone()
        graph.replay()
        torch.cuda.synchronize()
        got, qg, kg, vg = out.clone(), q_out.clone(), s.dk.clone(), s.dv.clone()
        s.dk.copy_(k0), s.dv.copy_(v0), out.zero_(), q_out.zero_()
        step()
        torch.cuda.synchronize()
        assert torch.equal(out, got) and torch.equal(q_out, qg) and torch.equal(s.dk, kg) and torch.equal(s.dv, vg)
        assert not got.isnan().any()


def test_two_graphs_and_a_grown_workspace():
    """Two graphs of one context, the second captured after a call that grew the workspace: replays in turn, with eager
    calls between, give each one's eager result."""
    c = N.Context(0)
    calls, graphs = [], []
    for i, (lengths, prefix) in enumerate([([(1, 2206)], None), ([(1, 900)] * 9, 4), ([(157, 2205), (1, 700)], None)]):
        s = Setup(F16, 128, 16, 8, 64, lengths, seed=110 + i, shared=prefix or 0)
        q, out = s.queries().cuda(), torch.zeros(s.rows, 16, 128, dtype=F16, device="cuda")
        s.attend(c, q, prefix=prefix, out=out)
        torch.cuda.synchronize()
        calls.append((s, q, out, prefix, out.clone()))
        if i < 2:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                s.attend(c, q, prefix=prefix, out=out)
            graphs.append(g)
    for turn in range(4):
        for i in (0, 1, 0):
            calls[i][2].zero_()
            graphs[i].replay()
            s, q, out, prefix, first = calls[2 if turn % 2 else 1 - i]
            s.attend(c, q, prefix=prefix, out=out)  # eager, behind it
            torch.cuda.synchronize()
            assert torch.equal(out, first) and torch.equal(calls[i][2], calls[i][4])
    del graphs
    c.close()


def test_a_refused_workspace_leaves_the_next_call_alone():
    """A call whose parts would need more memory than the card has (over a tebibyte) returns an error and runs nothing;
    the next call is as ever."""
    c = N.Context(0)
    s = Setup(F16, 256, 16, 8, 64, [(1, 300), (1, 200)], seed=120, shared=2)
    q = s.queries().cuda()
    ref, bound = s.expect(q.cpu())
    c.set_tuning("attn_mid", 0)
    c.set_tuning("attn_parts", 32)
    many = N.KvBatch(s.dtable, s.dstarts, s.dlen, 1 << 21, 1, s.max_kv)  # 2^25 rows, in 32 parts of 1 KiB each
    assert (1 << 25) * 32 * 1024 > 2 * torch.cuda.mem_get_info()[1]
    big = [torch.empty(1 << 21, 16, 256, dtype=F16, device="cuda") for _ in range(2)]
    with pytest.raises(N.NsError, match="memory"):
        c.shared_prefix_attention(s.cache, many, 2, big[0], 16, 1 / 16, big[1])
    del big
    torch.cuda.empty_cache()
    c.set_tuning("attn_mid", -1)
    c.set_tuning("attn_parts", 0)
    assert_within(s.attend(c, q, prefix=2), ref, bound)
    torch.cuda.synchronize()
    c.close()


def test_on_another_stream(ctx):
    s = Setup(F16, 256, 16, 8, 64, [(1, 3000), (20, 200)], seed=102)
    q = s.queries()
    dq = q.cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = s.attend(ctx, dq)
    b = None
    side.synchronize()
    b = s.attend(ctx, dq, stream=side.cuda_stream)
    side.synchronize()
    ref, bound = s.expect(q)
    assert_within(a, ref, bound)
    assert torch.equal(a, b)


def test_two_contexts_at_once():
    """Calls of two contexts that overlap on two streams do not disturb each other."""
    cs = [N.Context(0), N.Context(0)]
    ss = [Setup(F16, 256, 16, 8, 64, [(1, 4000)], seed=103 + i) for i in range(2)]
    qs = [s.queries() for s in ss]
    dq = [q.cuda() for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                outs[i].append(ss[i].attend(cs[i], dq[i]))
    torch.cuda.synchronize()
    for i in range(2):
        ref, bound = ss[i].expect(qs[i])
        assert_within(outs[i][0], ref, bound)
        for o in outs[i]:
            assert torch.equal(o, outs[i][0])
    for c in cs:
        c.close()


@pytest.mark.parametrize("dtype", [F16, E4M3], ids=["f16", "e4m3"])
def test_a_layer_as_an_engine_runs_it(ctx, dtype):
    """ns_qkv, ns_kv_append, ns_paged_attention and the output projection over a prompt in two chunks, single tokens
    and a verification step: what each step stores, and its attention on the cache as it then stands."""
    cols, qh, kh, D, page = 512, 4, 2, 64, 16
    steps = [40, 23, 1, 1, 3, 1]
    total = sum(steps)
    w = {name: torch.from_numpy(N.synth_weights(N.Q4_K, 110 + i, rows, c)).cuda()
         for i, (name, rows, c) in enumerate((("q", qh * D, cols), ("k", kh * D, cols), ("v", kh * D, cols), ("o", cols, qh * D)))}
    x = torch.from_numpy(N.synth_normal_f16(115, total * cols).view(np.int16)).view(total, cols).cuda()
    norm_q, norm_k = (1 + 0.1 * torch.randn(D, generator=torch.Generator().manual_seed(i)) for i in range(2))
    freqs = torch.from_numpy(N.rope_freqs(1e4, D)).cuda()
    nq, nk, nv = norm_q.cuda(), norm_k.cuda(), torch.ones(D, device="cuda")

    s = Setup(dtype, D, qh, kh, page, [(total, total)], seed=116)
    at = 0
    for n in steps:
        xi = x[at:at + n].contiguous()
        q, k, v = (torch.empty(n, h * D, device="cuda") for h in (qh, kh, kh))
        if n > 1:
            ctx.qkv(w["q"], w["k"], w["v"], N.Q4_K, N.ROW_MAJOR, cols, qh * D, kh * D, n, xi, q, k, v)
        else:  # one token takes fp32 input
            xf = xi.view(torch.float16).float()
            for name, y in (("q", q), ("k", k), ("v", v)):
                ctx.matmul(w[name], N.Q4_K, N.ROW_MAJOR, cols, y.shape[1], 1, xf, y)
        at += n
        s.lengths, s.T, s.rows = [(n, at)], n, n
        i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
        s.dstarts, s.dlen = i32(0, n), i32(at)
        s.batch = N.KvBatch(s.dtable, s.dstarts, s.dlen, n, n, at)
        q16 = torch.empty(n, qh, D, dtype=F16, device="cuda")
        ctx.kv_append(s.cache, s.batch, q, k, v, qh, freqs, D, q16, q_norm=nq, k_norm=nk, v_norm=nv)
        half = n > 1  # the output projection takes fp16 from 2 tokens on
        o = s.attend(ctx, q16, half_out=half)
        proj = torch.empty(n, cols, device="cuda")
        ctx.matmul(w["o"], N.Q4_K, N.ROW_MAJOR, qh * D, cols, n, o, proj, half_input=half)
        torch.cuda.synchronize()
        # the cache holds this step's keys and values: norm, turn and rounding of the projections
        pos = torch.arange(at - n, at)
        for cache, u, weight, turn, scale, values in ((s.dk, k, norm_k, True, s.ks, False), (s.dv, v, torch.ones(D), False, s.vs, True)):
            ref, mag = O.rotated(O.normed(u.cpu().view(n, kh, D), weight, 1e-6), pos, freqs.cpu(), D if turn else 0, False)
            err = (D / 2 + 24) * O.U32 * mag / scale
            step = (O.U16, 2.0 ** -25) if dtype == F16 else (O.U8, 2.0 ** -10)
            assert_within(O.read_new(cache.cpu(), s.table, [(n, at)], page, values).float(), ref / scale,
                          err + step[0] * (ref.abs() / scale + err) + step[1])
        s.k, s.v = s.dk.cpu(), s.dv.cpu()
        ref, bound = s.expect(q16.cpu(), half_out=half)
        assert_within(o, ref, bound)
        assert torch.isfinite(proj).all() and float(proj.abs().max()) > 0
