"""The 8-bit cache on the GPU: append byte for byte, attention against a plain computation in 64 bits."""
import math
import struct

import pytest
import torch

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture(scope="module")
def bk(lib):
    import bikv_pagecopy
    return bikv_pagecopy


class World:
    """A cache with ragged sequences on random pages, held on the host too."""

    def __init__(self, bk, cuda, lens, news, P=16, H=2, D=128, Hq=None, dtype="bf16", seed=0, spare=5, layers=2, ragged=True, pad=0, foreign=True, wide=0):
        g = torch.Generator().manual_seed(seed)
        self.P, self.H, self.D, self.Hq, self.t = P, H, D, Hq or H, TYPES[dtype]
        self.lens, self.news = list(lens), list(news)
        per = [-(-n // P) for n in lens]
        self.N = sum(per) + spare
        self.M = max(per + [1]) + 1 + -(-wide // P)         # columns of the page table: `wide` tokens more than any sequence has
        x = torch.randn((layers, 2, self.N, P, H, D), generator=g) * 60
        self.bytes = x.clamp(-448, 448).to(FP8).view(torch.uint8)
        self.scale = torch.exp2(torch.randint(-9, -5, (layers, 2, self.N, H), generator=g).float())
        if foreign:
            self.scale *= 0.7 + 0.6 * torch.rand(self.scale.shape, generator=g)
        ids = torch.randperm(self.N, generator=g)
        self.table = torch.full((len(lens), self.M), -7, dtype=torch.int64)
        at = 0
        for b, n in enumerate(per):
            self.table[b, :n] = ids[at:at + n]
            at += n
        starts = [pad]
        for n in self.news:
            starts.append(starts[-1] + n)
        self.starts = torch.tensor(starts)
        self.rows = starts[-1] + pad
        self.ragged = ragged
        self.payload_d, self.scale_d = self.bytes.to(cuda).view(FP8), self.scale.to(cuda)
        self.cache = bk.FP8KVCache(self.payload_d, self.scale_d)
        self.table_d, self.lens_d = self.table.to(cuda), torch.tensor(self.lens, device=cuda)
        self.starts_d = self.starts.to(cuda) if ragged else None
        self.g, self.cuda = g, cuda

    def push(self):
        """The host's bytes and scales (changed by a test) to the GPU."""
        self.payload_d.view(torch.uint8).copy_(self.bytes)
        self.scale_d.copy_(self.scale)

    def randn(self, heads, mul=1.0):
        return (torch.randn((self.rows, heads, self.D), generator=self.g) * mul).to(self.t)

    def append(self, k, v, layer=1):
        self.cache.append(layer, k.to(self.cuda), v.to(self.cuda), self.table_d, self.lens_d, self.starts_d)

    def attend(self, q, layer=1, **kw):
        return self.cache.attend(layer, q.to(self.cuda), self.table_d, self.lens_d, self.starts_d, return_lse=True, **kw)


# ---- append -------------------------------------------------------------------------------------
def _grid(x):
    """float64 -> nearest e4m3 value (ties to even), NaN kept."""
    mag = x.abs().clamp(min=2.0 ** -30)
    e = torch.floor(torch.log2(mag))
    e = torch.where(torch.exp2(e) > mag, e - 1, torch.where(torch.exp2(e + 1) <= mag, e + 1, e)).clamp(min=-6)
    step = torch.exp2(e - 3)
    return torch.where(x.isnan(), x, torch.round(x / step) * step)


def _needed(amax):
    s = 2.0 ** -126
    while 448 * s < amax:
        s *= 2
    return s


def _append_oracle(w, k, v, layer=1):
    """What the cache stands for after the append: (values [2, N, P, H, D] float64 before the scale, scales [2, N, H])."""
    vals = w.bytes[layer].view(FP8).double().clone()
    scales = w.scale[layer].double().clone()
    for b, (n, new) in enumerate(zip(w.lens, w.news)):
        for pos in sorted({p // w.P for p in range(n - new, n)}):
            lo, hi = max(n - new, pos * w.P), min(n, (pos + 1) * w.P)
            page, r0 = int(w.table[b, pos]), lo - pos * w.P
            t = int(w.starts[b]) + lo - (n - new)
            for kv, x in ((0, k), (1, v)):
                for h in range(w.H):
                    y = x[t:t + hi - lo, h].double()
                    y = torch.where(y.isinf(), torch.full_like(y, math.nan), y)
                    fin = y[~y.isnan()]
                    amax = float(fin.abs().max()) if fin.numel() else 0.0
                    old = float(scales[kv, page, h])
                    if r0 > 0 and 448 * old >= amax:
                        s = old
                    else:
                        s = _needed(amax)
                        if r0 > 0:
                            # the product is rounded to fp32 before it is rounded to e4m3, as the definition's fp32 arithmetic does
                            prod = (vals[kv, page, :r0, h].float() * torch.tensor(old, dtype=torch.float32)).double()
                            vals[kv, page, :r0, h] = _grid(prod / s)
                    scales[kv, page, h] = s
                    quo = y * 0 if s == 0 else (y.float() / torch.tensor(s, dtype=torch.float32)).double()
                    vals[kv, page, r0:r0 + hi - lo, h] = _grid(quo)
    return vals, scales


def _check_append(w, k, v, layer=1):
    vals, scales = _append_oracle(w, k, v, layer)
    other = 1 - layer
    w.append(k, v, layer)
    w.cache.check()
    got = w.payload_d.cpu()
    assert torch.equal(w.scale_d[layer].cpu().double(), scales)
    assert torch.equal(got[other].view(torch.uint8), w.bytes[other]) and torch.equal(w.scale_d[other].cpu(), w.scale[other])
    have = got[layer].double()
    assert torch.equal(have.isnan(), vals.isnan())
    assert torch.equal(have.nan_to_num(), vals.nan_to_num())
    # rows behind the new tokens, and pages of nobody, keep their bytes
    kept = torch.ones(w.N, w.P, dtype=torch.bool)
    for b, n in enumerate(w.lens):
        for p in range(n):
            kept[int(w.table[b, p // w.P]), p % w.P] = False
    assert torch.equal(got[layer].view(torch.uint8)[:, kept], w.bytes[layer][:, kept])


APPENDS = [
    # lens (new tokens included), new tokens
    ([1], [1]), ([17], [1]), ([16], [16]), ([5, 33, 64], [5, 1, 64]), ([100, 31, 7, 250], [37, 31, 2, 190]), ([40, 40], [0, 40]), ([129], [129]),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("P,H,D", [(16, 2, 128), (1, 3, 64), (50, 4, 128), (32, 8, 64), (70, 1, 128), (7, 5, 64)])
@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append(bk, cuda, case, P, H, D, dtype):
    lens, news = APPENDS[case]
    w = World(bk, cuda, lens, news, P=P, H=H, D=D, dtype=dtype, seed=case, pad=case % 3)
    _check_append(w, w.randn(H, 3.0), w.randn(H, 0.02))


@pytest.mark.parametrize("mul", [0.0, 1e-7, 1e-3, 1.0, 40.0, 6000.0])
def test_append_keeps_or_grows_the_scale_of_a_page_with_older_tokens(bk, cuda, mul):
    w = World(bk, cuda, [9, 26, 31], [3, 1, 14], seed=3)
    _check_append(w, w.randn(2, mul), w.randn(2, mul))


def test_append_of_extreme_values(bk, cuda):
    w = World(bk, cuda, [20, 16, 3, 40, 24], [20, 16, 3, 40, 20], dtype="bf16", seed=4)
    k, v = w.randn(2), w.randn(2)
    k[0] = 3.3e38                                  # next to the largest value
    k[1, :, ::2] = -3.3e38
    k[21] = 0.0
    v[20:36] = 0.0                                 # a whole page of zeros
    k[36:39] = 1e-39                               # subnormal in bf16
    k[40, 0, 5], k[41, 1, 6], v[42, 0, 7] = math.nan, math.inf, -math.inf
    v[50] = math.nan                               # every value of a token
    _check_append(w, k, v)


def test_append_at_the_edge_of_each_power_of_two(bk, cuda):
    """448 s is held, the next value is not."""
    vals = [448.0, 450.0, 446.0, 1.75, 1.7578125, 1.7421875, 896.0, 900.0, 2.0, 1.0]
    w = World(bk, cuda, [1] * len(vals), [1] * len(vals), P=4, H=1, dtype="bf16", seed=5)
    k = torch.zeros(len(vals), 1, 128, dtype=torch.bfloat16)
    for i, x in enumerate(vals):
        k[i, 0, i] = x
    _check_append(w, k, -k)


def test_append_over_odd_old_scales(bk, cuda):
    """A cache filled elsewhere: zero, subnormal, infinite and huge scales of a page that already holds tokens."""
    w = World(bk, cuda, [6] * 6, [2] * 6, P=8, H=1, seed=6)
    for b, s in enumerate([0.0, 1e-40, 2.0 ** 127, 1e-3, 3.0, 2.0 ** -126]):
        w.scale[1, :, int(w.table[b, 0])] = s
    w.push()
    k = w.randn(1)
    k[0:2] = 0.0                                   # the zero scale is kept where the new values are zero, too
    _check_append(w, k, k.clone())


def test_one_token_at_a_time_stays_as_first_rounded(bk, cuda):
    """Appending token by token gives what appending at once gives, but for the scale's history: every token is within
    half a step of its value at the page's last scale."""
    w = World(bk, cuda, [16], [1], seed=7)
    x = w.randn(2)[:1].repeat(16, 1, 1) * torch.linspace(0.1, 9, 16)[:, None, None].to(w.t)
    for n in range(1, 17):
        w.lens_d.fill_(n)
        w.cache.append(1, x[n - 1:n].to(cuda), x[n - 1:n].to(cuda), w.table_d, w.lens_d, None)
    w.cache.check()
    page = int(w.table[0, 0])
    s = w.scale_d[1, :, page].cpu().double()
    got = w.payload_d[1, :, page].cpu().double() * s[:, None, :, None]
    # a normal e4m3 value is off by 2^-4 of itself at most; below the normal range by half the smallest step, twice over (both roundings)
    tol = x.double().abs() * 2.0 ** -4 + s.max() * 2.0 ** -9
    assert ((got - x.double()).abs() <= tol).all()


def test_append_takes_strided_rows_and_leaves_rows_of_nobody(bk, cuda):
    w = World(bk, cuda, [30, 12], [13, 12], H=2, D=128, seed=8, pad=4)
    fused = torch.randn((w.rows, 10, 128), generator=w.g).to(w.t)      # q, k, v of one projection side by side
    k, v = fused[:, 6:8], fused[:, 8:10]
    vals, scales = _append_oracle(w, k, v)
    f = fused.to(cuda)
    w.cache.append(1, f[:, 6:8], f[:, 8:10], w.table_d, w.lens_d, w.starts_d)
    w.cache.check()
    assert torch.equal(w.payload_d[1].cpu().double(), vals) and torch.equal(w.scale_d[1].cpu().double(), scales)
    # heads outermost
    w.push()
    kt = k.transpose(0, 1).contiguous().to(cuda).transpose(0, 1)
    w.cache.append(1, kt, f[:, 8:10], w.table_d, w.lens_d, w.starts_d)
    w.cache.check()
    assert torch.equal(w.payload_d[1].cpu().double(), vals)


def test_append_skips_what_makes_no_sense_and_says_so(bk, cuda):
    lens, news = [20, 18, 25, 30], [4, 4, 4, 4]
    for spoil in ("len", "negative", "more rows than tokens", "page", "negative page", "starts"):
        w = World(bk, cuda, lens, news, seed=9)
        k, v = w.randn(2), w.randn(2)
        good = [0, 2, 3]
        if spoil == "len":
            w.lens_d[1] = w.M * w.P + 1
        elif spoil == "negative":
            w.lens_d[1] = -3
        elif spoil == "more rows than tokens":
            w.lens_d[1] = 2
        elif spoil == "page":
            w.table_d[1, 1] = w.N
        elif spoil == "negative page":
            w.table_d[1, 1] = -1
        else:
            w.starts_d[4] = w.rows + 1
            good = [0, 1, 2]
        bad = ({0, 1, 2, 3} - set(good)).pop()
        vals, scales = _append_oracle(w, k, v)
        w.append(k, v)
        with pytest.raises(RuntimeError, match="page-id" if "page" in spoil else "source-range"):
            w.cache.check()
        got, gs = w.payload_d[1].cpu(), w.scale_d[1].cpu()
        for b in good:
            p = w.table[b, :-(-lens[b] // w.P)]
            assert torch.equal(got.double()[:, p], vals[:, p]) and torch.equal(gs.double()[:, p], scales[:, p]), (spoil, b)
        p = w.table[bad, 1:2]
        if spoil != "more rows than tokens":
            assert torch.equal(got.view(torch.uint8)[:, p], w.bytes[1][:, p]), spoil
        w.cache.check()


# ---- attention ----------------------------------------------------------------------------------
def _attend_oracle(w, q, causal=True, scale=None, layer=1):
    """(out, lse, tolerance of out, tolerance of lse), float64. With p the softmax's terms, A = sum p |v| / sum p and S a row's
    largest sum of |scale q k|: the kernel rounds p to fp16 (2^-11 of it; below fp16's normal range, 2^-33 of the largest
    possible p, in units of the largest V scale, which a factor 2 covers), sums D products and then n keys in fp32
    (2^-24 each, as a share of what is summed), and takes exp2 and log2 to about 2^-22; the output's own rounding is eps / 2."""
    D, G, P = w.D, w.Hq // w.H, w.P
    scale = 1 / math.sqrt(D) if scale is None else scale
    val = w.bytes[layer].view(FP8).double() * w.scale[layer].double()[:, :, None, :, None]
    out = torch.zeros((w.rows, w.Hq, D), dtype=torch.float64)
    lse = torch.full((w.rows, w.Hq), -math.inf, dtype=torch.float64)
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    eps = torch.finfo(w.t).eps
    for b, (n, new) in enumerate(zip(w.lens, w.news)):
        pages = w.table[b, :-(-n // P)]
        ok = ((pages >= 0) & (pages < w.N)).repeat_interleave(P)[:n]
        kv = val[:, pages.clamp(0, w.N - 1)].reshape(2, -1, w.H, D)[:, :n]
        vs = w.scale[layer, 1][pages.clamp(0, w.N - 1)].double()
        r = slice(int(w.starts[b]), int(w.starts[b]) + new)
        if not new:
            continue
        for h in range(w.Hq):
            k, v = kv[0, :, h // G], kv[1, :, h // G]
            x = q[r, h].double()
            z = x @ k.t() * scale
            S = (x.abs() @ k.abs().t() * abs(scale))
            see = ok[None].expand(new, n).clone()
            if causal:
                see &= torch.arange(n)[None] <= (n - new + torch.arange(new))[:, None]
            z = torch.where(see, z, torch.full_like(z, -math.inf))
            if n == 0:
                continue
            any_ = see.any(1)
            lse[r, h] = torch.logsumexp(z, 1)
            p = torch.where(see, torch.exp(z - torch.where(any_, lse[r, h], torch.zeros_like(lse[r, h]))[:, None]), torch.zeros_like(z))
            vz = torch.where(see[:, :, None] if v.isnan().any() else torch.ones(1, dtype=torch.bool), v[None], torch.zeros(1, dtype=torch.float64)) if v.isnan().any() else None
            out[r, h] = (p[:, :, None] * vz).sum(1) if vz is not None else p @ v
            A = p @ v.nan_to_num().abs()
            dz = (D + 4) * 2.0 ** -24 * torch.where(see, S, torch.zeros_like(S)).nan_to_num().amax(1)
            tiny = n * 448 * 2 * float(vs[:, h // G][vs[:, h // G].isfinite()].abs().max() if vs.numel() else 0) * 2.0 ** -33
            tol[r, h] = eps / 2 * out[r, h].abs() + A * (2.0 ** -11 + 2 * dz[:, None] + 2.0 ** -21 + (n + 8) * 2.0 ** -24) + tiny
            ltol[r, h] = dz + 2.0 ** -21 * (1 + torch.where(any_, lse[r, h].abs(), torch.zeros_like(dz))) + (n + 8) * 2.0 ** -24
    return out, lse, tol, ltol


def _compare(w, q, got, causal=True, scale=None, layer=1):
    out, lse, tol, ltol = _attend_oracle(w, q, causal, scale, layer)
    rows = slice(int(w.starts[0]), int(w.starts[-1]))
    o, l = got[0].cpu().double()[rows], got[1].cpu().double()[rows]
    out, lse, tol, ltol = out[rows], lse[rows], tol[rows], ltol[rows]
    assert torch.equal(o.isnan(), out.isnan())
    fine = ~out.isnan()
    over = ((o - out).abs() - tol)[fine]
    assert not (over > 0).any(), f"out is off by {float(over.max())} more than it may be"
    none = lse == -math.inf
    assert torch.equal(l == -math.inf, none) and not o[none].nan_to_num(nan=1.0).any()
    seen = ~none & ~lse.isnan()
    assert ((l - lse).abs() <= ltol)[seen].all()


def _run(w, q, **kw):
    got = w.attend(q, **kw)
    w.cache.check()
    kw.pop("out", None)
    _compare(w, q, got, causal=kw.get("causal", True), scale=kw.get("softmax_scale"))
    return got


ATTENDS = [
    # lens, new tokens, q heads per KV head
    ([1], [1], 1),
    ([63, 64, 65, 1, 128, 200], [1] * 6, 4),
    ([777], [1], 6),
    ([3000, 5, 0, 129], [1, 1, 1, 1], 7),
    ([90, 300], [5, 3], 7),                        # 21 to 35 rows
    ([200, 33, 70], [2, 33, 0], 8),
    ([131], [131], 1),
    ([400, 257, 90], [300, 128, 90], 2),           # many rows
    ([1100], [260], 4),
    ([7, 3], [9, 5], 2),                           # more rows than keys: the first see nothing
    ([0, 0], [2, 1], 1),
    ([150, 10], [160, 200], 1),
    ([40] * 70, [1] * 70, 2),                      # more sequences than a wave has lanes
    ([5 + i % 40 for i in range(300)], [i % 3 for i in range(300)], 3),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("P,H,D", [(16, 2, 128), (50, 1, 128), (1, 3, 64), (32, 8, 64), (8, 2, 128)])
@pytest.mark.parametrize("case", range(len(ATTENDS)))
def test_attend(bk, cuda, case, P, H, D, dtype):
    lens, news, G = ATTENDS[case]
    if sum(lens) * H > 12000:
        H = 1
    # every other world has a table with room for long sequences, which cuts the same work another way
    w = World(bk, cuda, lens, news, P=P, H=H, D=D, Hq=G * H, dtype=dtype, seed=case, ragged=any(n != 1 for n in news) or case % 2 == 0,
              wide=9000 * ((case + P + (dtype == "bf16")) % 2))
    _run(w, w.randn(w.Hq, 1.5), causal=True)
    _run(w, w.randn(w.Hq, 1.5), causal=False)


SHAPES = [
    # lens, new tokens (None: one each, without row numbers), KV heads, q heads per KV head, head size
    ([70, 300, 5], None, 2, 40, 128),                                # one token, more rows than a narrow tile has
    ([500, 130], None, 1, 200, 64),                                  # and more than a wide one has
    ([600, 64, 33, 9], [5, 8, 6, 7], 2, 8, 128),                     # 40 to 64 rows
    ([100 + 4 * i for i in range(33)], [5 + i % 4 for i in range(33)], 4, 8, 64),
    ([5 + 3 * i for i in range(60)], None, 9, 2, 64),                # heads that do not fill their workgroups
    ([200, 77], None, 12, 1, 128),
    ([200, 77], [2, 3], 17, 5, 64),
    ([40] * 53, [1 + i % 2 for i in range(53)], 4, 8, 128),          # as many workgroups as CUs, and more
    ([30 + i for i in range(130)], None, 3, 6, 64),
    ([90 + 41 * i for i in range(10)], [5 - i % 5 for i in range(10)], 2, 7, 128),        # 7 to 35 rows, eight sequences and more
    ([20 + 50 * i for i in range(9)], None, 3, 32, 64),
    ([700 - 60 * i for i in range(10)], [2 + i % 2 for i in range(10)], 9, 8, 64),
    ([1500, 3, 0, 800, 64, 65, 1, 31], [4, 3, 0, 4, 4, 1, 1, 5], 2, 8, 128),
    ([1024, 1000], None, 2, 4, 128), ([1025, 17], None, 2, 4, 128),  # either side of the length from which work is cut
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("wide", [0, 9000])
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_attend_whichever_way_the_work_is_cut(bk, cuda, case, wide, dtype):
    lens, news, H, G, D = SHAPES[case]
    w = World(bk, cuda, lens, news or [1] * len(lens), P=16, H=H, D=D, Hq=G * H, dtype=dtype, seed=50 + case, ragged=news is not None, wide=wide)
    _run(w, w.randn(w.Hq, 1.5), causal=True)
    _run(w, w.randn(w.Hq, 1.5), causal=False)


def test_row_numbers_that_fall_and_overlap_do_no_harm(bk, cuda):
    """Sequences whose rows make no sense are skipped and reported; those whose rows are others', too, may hold either's result."""
    for lens, starts in (([300, 40, 300], [0, 20, 5, 25]), ([70, 70, 70, 70], [0, 9, 0, 9, 0]), ([3000, 3000, 10], [0, 25, 0, 25])):
        for wide in (0, 9000):
            w = World(bk, cuda, lens, [1] * len(lens), H=2, Hq=8, seed=70, wide=wide)
            w.rows = max(starts)
            q = w.randn(8).to(cuda)
            k = w.randn(2).to(cuda)
            s = torch.tensor(starts, device=cuda)
            w.cache.attend(1, q, w.table_d, w.lens_d, s)
            with pytest.raises(RuntimeError):
                w.cache.check()
            w.cache.append(1, k, k, w.table_d, w.lens_d, s)
            with pytest.raises(RuntimeError):
                w.cache.check()
    w = World(bk, cuda, [100, 20], [3, 1], H=2, Hq=8, seed=71)
    q = w.randn(8)
    _run(w, q)                                                       # and the next call is none the worse


def test_tensors_that_want_a_gradient_are_refused(bk, cuda):
    w = World(bk, cuda, [40, 20], [1, 1], H=2, Hq=4, seed=72, ragged=False)
    k, q = w.randn(2).to(cuda), w.randn(4).to(cuda)
    wants = lambda x: x.clone().requires_grad_()
    for bad in (lambda: w.cache.attend(1, wants(q), w.table_d, w.lens_d), lambda: w.cache.append(1, wants(k), k, w.table_d, w.lens_d),
                lambda: w.cache.append(1, k, wants(k), w.table_d, w.lens_d), lambda: w.cache.attend(1, q, w.table_d, w.lens_d, out=wants(q))):
        with pytest.raises(RuntimeError, match="gradient"):
            bad()
    with torch.no_grad():
        w.cache.append(1, wants(k), k, w.table_d, w.lens_d)
        w.cache.attend(1, wants(q), w.table_d, w.lens_d)
    w.cache.check()


def test_the_softmax_scale_and_peaked_rows(bk, cuda):
    for scale in (0.0, -0.3, 0.02, 2.0):
        w = World(bk, cuda, [300, 77], [1, 4], H=2, Hq=8, seed=20)
        _run(w, w.randn(8), softmax_scale=scale)
        w = World(bk, cuda, [300], [150], H=1, Hq=2, seed=21)
        _run(w, w.randn(2), softmax_scale=scale)


def test_pages_whose_v_scales_lie_far_apart(bk, cuda):
    for lens, news in (([700, 300], [1, 3]), ([700], [200])):
        w = World(bk, cuda, lens, news, H=2, Hq=4, seed=22)
        e = torch.randint(-100, 60, w.scale[1, 1].shape, generator=w.g).double()
        w.scale[1, 1] = torch.exp2(e).float() * w.scale[1, 1]
        w.scale[1, 1, ::5] = 0.0
        w.push()
        _run(w, w.randn(4))


@pytest.mark.parametrize("lens,news", [([100, 37, 300], [1, 1, 1]), ([100, 37, 300], [4, 7, 2]), ([333, 200], [333, 130])])
@pytest.mark.parametrize("wide", [0, 9000])
@pytest.mark.parametrize("causal", [True, False])
def test_nothing_behind_a_sequence_reaches_it(bk, cuda, lens, news, causal, wide):
    """Bytes behind the last token, spare pages and their scales are NaN or infinite."""
    w = World(bk, cuda, lens, news, H=2, Hq=8, seed=23, wide=wide)
    mine = torch.zeros(w.N, w.P, dtype=torch.bool)
    for b, n in enumerate(lens):
        for p in range(n):
            mine[int(w.table[b, p // w.P]), p % w.P] = True
    w.bytes[1][:, ~mine] = 0x7f
    w.bytes[1][:, ~mine, :, ::2] = 0xff
    spare = ~mine.any(1)
    w.scale[1][:, spare] = math.nan
    w.scale[1, 0][spare] = math.inf
    w.push()
    _run(w, w.randn(8), causal=causal)


@pytest.mark.parametrize("wide", [0, 9000])
@pytest.mark.parametrize("G,news", [(1, [6]), (4, [12]), (8, [7]), (2, [130])])
def test_nan_of_a_later_token_stays_out_of_earlier_rows(bk, cuda, G, news, wide):
    """A token whose K or V is NaN: the rows before it do not see it; the rows from it on get NaN where V is NaN, and everywhere where K is."""
    w = World(bk, cuda, [200], news, H=1, Hq=G, seed=24, wide=wide)
    bad = 200 - news[0] + news[0] // 2
    page, row = int(w.table[0, bad // w.P]), bad % w.P
    w.bytes[1, 1, page, row, 0, 3] = 0x7f
    w.bytes[1, 1, page, row, 0, 77] = 0xff
    w.push()
    q = w.randn(G)
    got = _run(w, q)
    o = got[0].cpu().float()
    first = news[0] // 2
    assert not o[:first].isnan().any() and o[first:, :, [3, 77]].isnan().all()
    w.bytes[1, 0, page, row, 0, 9] = 0x7f
    w.push()
    got = w.attend(q)
    w.cache.check()
    o, l = got[0].cpu().float(), got[1].cpu()
    assert not o[:first].isnan().any() and o[first:].isnan().all() and l[first:].isnan().all() and not l[:first].isnan().any()


@pytest.mark.parametrize("news", [[20], [140]])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_a_page_scale_that_is_not_finite_spoils_only_rows_that_see_the_page(bk, cuda, news, value):
    w = World(bk, cuda, [208], news, P=16, H=1, Hq=2, seed=25)
    w.bytes[1][:, int(w.table[0, 12])] |= 0x08                     # no zero among its bytes: 0 * inf would hide nothing
    w.scale[1, 1, int(w.table[0, 12])] = value                     # tokens 192 .. 207
    w.push()
    got = w.attend(w.randn(2))
    w.cache.check()
    o = got[0].cpu().float()
    first = 192 - (208 - news[0])
    assert o[:first].isfinite().all() and not o[first:].isfinite().any()


def test_a_bad_page_is_left_out_and_reported(bk, cuda):
    for lens, news in (([200, 90], [1, 1]), ([200, 90], [9, 3]), ([400, 90], [300, 20])):
        w = World(bk, cuda, lens, news, H=2, Hq=4, seed=26, wide=9000 * (news[0] == 1))
        w.table[0, 2], w.table[0, 5], w.table[1, 0] = -1, w.N, 1 << 40
        w.table_d.copy_(w.table)
        q = w.randn(4)
        got = w.attend(q)
        with pytest.raises(RuntimeError, match="page-id"):
            w.cache.check()
        _compare(w, q, got)


def test_a_sequence_that_makes_no_sense_is_skipped_and_reported(bk, cuda):
    for lens, news in (([200, 90, 50], [1, 1, 1]), ([200, 90, 50], [2, 3, 1]), ([400, 300, 250], [300, 250, 200])):
        for spoil in ("long", "negative"):
            w = World(bk, cuda, lens, news, H=2, Hq=4, seed=27, wide=9000 * (spoil == "long"))
            q = w.randn(4)
            out = torch.full((w.rows, 4, 128), 7.0, dtype=w.t, device=cuda)
            w.lens_d[1] = -1 if spoil == "negative" else w.M * w.P + 1
            got = w.attend(q, out=out)
            with pytest.raises(RuntimeError, match="source-range"):
                w.cache.check()
            assert got[0].data_ptr() == out.data_ptr()
            want, _, tol, _ = _attend_oracle(w, q)
            o = out.cpu().double()
            a, b = int(w.starts[1]), int(w.starts[2])
            assert (o[a:b] == 7.0).all()
            for r in (slice(0, a), slice(b, w.rows)):
                assert ((o[r] - want[r]).abs() <= tol[r]).all()


def test_rows_of_nobody_are_left_as_they_were(bk, cuda):
    for lens, news in (([70, 300], [1, 2]), ([400, 200], [150, 140])):
        w = World(bk, cuda, lens, news, H=2, Hq=4, seed=28, pad=3)
        q = w.randn(4)
        q[:3], q[-3:] = math.nan, math.nan
        out = torch.full((w.rows, 4, 128), 5.0, dtype=w.t, device=cuda)
        _run(w, q, out=out)
        assert (out[:3] == 5.0).all() and (out[-3:] == 5.0).all()


def test_strided_q_out_and_table(bk, cuda):
    for lens, news in (([70, 300], [1, 2]), ([400, 200], [150, 140])):
        w = World(bk, cuda, lens, news, H=2, Hq=6, seed=29)
        fused = torch.randn((w.rows, 10, 128), generator=w.g).to(w.t)
        q = fused[:, 2:8]
        buf = torch.full((6, w.rows, 128), 9.0, dtype=w.t, device=cuda)       # heads outermost
        wide = torch.full((len(lens), w.M + 5), -1, device=cuda)
        wide[:, 2:2 + w.M] = w.table_d
        got = w.cache.attend(1, fused.to(cuda)[:, 2:8], wide[:, 2:2 + w.M], w.lens_d, w.starts_d, out=buf.transpose(0, 1), return_lse=True)
        w.cache.check()
        _compare(w, q, got)


def test_the_same_call_gives_the_same_bits(bk, cuda):
    for lens, news in (([3000, 50, 700], [1, 1, 1]), ([1200, 800], [4, 3]), ([900], [260]), ([9000], [260])):
        w = World(bk, cuda, lens, news, H=2, Hq=8, seed=30)
        q = w.randn(8)
        a, b = w.attend(q), w.attend(q)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_parts_merge_by_their_lse(bk, cuda):
    """A shared prefix and a sequence's own pages attended apart and merged give what one call gives."""
    w = World(bk, cuda, [160 + 75], [1], H=2, Hq=8, seed=31)
    q = w.randn(8)
    whole = w.attend(q)
    one = w.cache.attend(1, q.to(cuda), w.table_d[:, :10].contiguous(), torch.tensor([160], device=cuda), None, causal=False, return_lse=True)
    two = w.cache.attend(1, q.to(cuda), w.table_d[:, 10:].contiguous(), torch.tensor([75], device=cuda), None, causal=False, return_lse=True)
    w.cache.check()
    lse = torch.logaddexp(one[1], two[1])
    out = one[0].double() * torch.exp(one[1] - lse).double()[..., None] + two[0].double() * torch.exp(two[1] - lse).double()[..., None]
    _, _, tol, ltol = _attend_oracle(w, q)
    # three roundings to the output's type take part: the two parts' and the whole call's
    eps = torch.finfo(w.t).eps
    part = (one[0].double().abs() + two[0].double().abs()).cpu() * eps / 2
    assert ((out - whole[0].double()).abs().cpu() <= 3 * tol + part).all()
    assert ((lse - whole[1]).abs().cpu() <= 3 * ltol).all()


def test_append_then_attend_as_a_step(bk, cuda):
    """Prompts of two sequences, then single tokens: each step writes and reads; the oracle follows the cache's bytes."""
    w = World(bk, cuda, [40, 23], [40, 23], H=2, Hq=8, seed=32, foreign=False)
    for step in range(4):
        if step:
            w.lens, w.news = [n + 1 for n in w.lens], [1, 1]
            w.starts = torch.tensor([0, 1, 2])
            w.rows = 2
            w.lens_d.add_(1)
            w.starts_d = None
        k, v, q = w.randn(2), w.randn(2), w.randn(8)
        vals, scales = _append_oracle(w, k, v)
        w.append(k, v)
        got = w.attend(q)
        w.cache.check()
        w.bytes, w.scale = w.payload_d.cpu().view(torch.uint8), w.scale_d.cpu()
        assert torch.equal(w.bytes[1].view(FP8).double(), vals) and torch.equal(w.scale[1].double(), scales)
        _compare(w, q, got)


@pytest.mark.parametrize("lens,news,G", [([500, 90, 33], [1, 1, 1], 4), ([300, 80], [3, 5], 6), ([700, 300], [200, 140], 2)])
def test_replays_from_a_graph_with_other_lengths(bk, cuda, lens, news, G):
    """One step captured; lengths, tokens and pages change between the replays, eager work runs in between."""
    w = World(bk, cuda, lens, news, H=2, Hq=2 * G, seed=33, foreign=False, spare=20, wide=9000 * (G == 4))
    k, v, q = (w.randn(h).to(cuda) for h in (2, 2, 2 * G))
    w.cache.append(1, k, v, w.table_d, w.lens_d, w.starts_d)
    w.cache.attend(1, q, w.table_d, w.lens_d, w.starts_d)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        w.cache.append(1, k, v, w.table_d, w.lens_d, w.starts_d)
        out, lse = w.cache.attend(1, q, w.table_d, w.lens_d, w.starts_d, return_lse=True)
    for i in range(4):
        w.lens = [max(n, m - 17 * i) for n, m in zip(news, lens)]
        w.lens_d.copy_(torch.tensor(w.lens))
        for x in (k, v, q):
            x.normal_()
        w.push()
        kh, vh, qh = k.cpu(), v.cpu(), q.cpu()
        vals, scales = _append_oracle(w, kh, vh)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        was = w.bytes, w.scale
        w.bytes, w.scale = w.payload_d.cpu().view(torch.uint8), w.scale_d.cpu()
        assert torch.equal(w.bytes[1].view(FP8).double(), vals) and torch.equal(w.scale[1].double(), scales)
        _compare(w, qh, (out, lse))
        eager = w.cache.attend(1, q, w.table_d, w.lens_d, w.starts_d, return_lse=True)
        assert torch.equal(eager[0], out) and torch.equal(eager[1], lse)
        w.bytes, w.scale = was
    w.cache.check()


def test_two_calls_at_once_on_two_streams(bk, cuda):
    w = World(bk, cuda, [5000, 700], [1, 1], H=2, Hq=8, seed=34)
    qs = [w.randn(8).to(cuda) for _ in range(2)]
    want = [w.cache.attend(1, q, w.table_d, w.lens_d) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(w.cache.attend(1, qs[i], w.table_d, w.lens_d))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_planes_beyond_4_gib(bk, cuda):
    """Byte offsets inside a plane pass 32 bits: pages of both calls lie behind them."""
    P, H, D, N = 64, 8, 128, 70000
    planes = [torch.empty((N, P, H, D), dtype=FP8, device=cuda) for _ in range(2)]
    scales = [torch.empty((N, H), device=cuda) for _ in range(2)]
    cache = bk.FP8KVCache.from_planes(planes, scales)
    for n, rows in ((200, 200), (200, 1), (130, 3)):
        ids = [69999, 65535, 65536, 3]
        table = torch.tensor([ids], device=cuda)
        k, v = (torch.randn(rows, H, D, device=cuda).bfloat16() for _ in range(2))
        q = torch.randn(rows, 2 * H, D, device=cuda).bfloat16()
        starts = torch.tensor([0, rows], device=cuda)
        lens = torch.tensor([n], device=cuda)
        cache.append(0, k, v, table, lens, starts)
        got = cache.attend(0, q, table, lens, starts, return_lse=True)
        cache.check()
        # the same on a small cache that holds copies of these pages (one page of a token slot more, never read)
        small = bk.FP8KVCache.from_planes([t[ids].contiguous() for t in (p.view(torch.uint8) for p in planes)], [s[ids].contiguous() for s in scales])
        t4 = torch.arange(4, device=cuda)[None]
        want = small.attend(0, q, t4, lens, starts, return_lse=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        small.append(0, k, v, t4, lens, starts)
        assert torch.equal(small.pool._keepalive[0][0], planes[0].view(torch.uint8)[ids])
        cache.check()


def test_the_pool_beside_the_cache_moves_its_pages(bk, cuda):
    """A fork: the parent's partly filled last page is copied inside the pool, with its scales, and both go on apart."""
    w = World(bk, cuda, [40], [1], H=2, Hq=4, seed=35, spare=3)
    free = [p for p in range(w.N) if p not in w.table[0, :3].tolist()]
    w.cache.pool.copy_pages(*w.cache.pool.page_moves([int(w.table[0, 2])], [free[0]]))
    child = w.table_d.clone()
    child[0, 2] = free[0]
    q = w.randn(4).to(cuda)
    a = w.cache.attend(1, q, w.table_d, w.lens_d)
    b = w.cache.attend(1, q, child, w.lens_d)
    assert torch.equal(a, b)
    batch = w.cache.pool.make_batch([w.table[0, :3].tolist()])
    staging, scales = w.cache.pool.gather(batch)
    w.cache.check()
    assert torch.equal(staging.view(4, 3, -1)[3].cpu(), w.bytes[1, 1][w.table[0, :3]].reshape(3, -1))
    assert torch.equal(scales.view(torch.float32).view(4, 3, -1)[3].cpu(), w.scale[1, 1][w.table[0, :3]])


def test_refusals(bk, lib, cuda):
    from bikv_pagecopy import _lib
    w = World(bk, cuda, [40, 20], [1, 1], H=2, Hq=4, seed=36, ragged=False)
    k, q = w.randn(2).to(cuda), w.randn(4).to(cuda)
    t, l = w.table_d, w.lens_d
    for bad in (lambda: w.cache.append(2, k, k, t, l), lambda: w.cache.append(-1, k, k, t, l),
                lambda: w.cache.append(1, k.float(), k.float(), t, l), lambda: w.cache.append(1, k, k.half(), t, l),
                lambda: w.cache.append(1, k[:1], k[:1], t, l), lambda: w.cache.append(1, k, k[:, :1], t, l),
                lambda: w.cache.append(1, k.cpu(), k, t, l), lambda: w.cache.append(1, k, k, t.int(), l),
                lambda: w.cache.append(1, k, k, t[:1], l), lambda: w.cache.append(1, k, k, t, l, torch.tensor([0, 2], device=cuda)),
                lambda: w.cache.append(1, k, k, t.t().contiguous().t(), l), lambda: w.cache.append(1, k, k, t.cpu(), l),
                lambda: w.cache.append(1, k.transpose(1, 2).contiguous().transpose(1, 2), k, t, l),
                lambda: w.cache.append(1, torch.randn(2, 2, 132, device=cuda).bfloat16()[..., 4:], k, t, l),     # not 16-byte aligned
                lambda: w.cache.attend(1, q[:, :3], t, l), lambda: w.cache.attend(1, q[..., :64], t, l),
                lambda: w.cache.attend(1, q.float(), t, l), lambda: w.cache.attend(1, q, t, l, softmax_scale=math.inf),
                lambda: w.cache.attend(1, q, t, l, softmax_scale=math.nan), lambda: w.cache.attend(1, q, t, l, out=q),
                lambda: w.cache.attend(1, q, t, l, out=q.half()), lambda: w.cache.attend(1, q, t, l, out=torch.empty(1, 4, 128, device=cuda).bfloat16().expand(2, 4, 128)),
                lambda: w.cache.attend(1, q[:, :0], t, l), lambda: w.cache.attend(1, q, t, l.int())):
        with pytest.raises(RuntimeError):
            bad()
    # nothing to do is no error
    none = torch.empty((0, 4, 128), dtype=torch.bfloat16, device=cuda)
    out = w.cache.attend(1, none, t[:0], l[:0])
    assert out.shape == none.shape
    w.cache.append(1, none[:, :2], none[:, :2], t[:0], l[:0])
    w.cache.append(1, none[:, :2], none[:, :2], t, l, torch.zeros(3, dtype=torch.int64, device=cuda))
    w.cache.attend(1, none, t, l, torch.zeros(3, dtype=torch.int64, device=cuda))
    # a table without columns: every sequence is empty
    out, lse = w.cache.attend(1, q, t[:, :0], torch.zeros_like(l), return_lse=True)
    w.cache.check()
    assert not out.any() and (lse == -math.inf).all()
    for make in (lambda: bk.FP8KVCache(w.payload_d[:, :1], w.scale_d), lambda: bk.FP8KVCache(w.payload_d, w.scale_d[:, :, :1]),
                 lambda: bk.FP8KVCache(w.payload_d, w.scale_d.half()), lambda: bk.FP8KVCache(w.payload_d.half(), w.scale_d),
                 lambda: bk.FP8KVCache(w.payload_d[..., :96].contiguous(), w.scale_d), lambda: bk.FP8KVCache(w.payload_d.cpu(), w.scale_d.cpu()),
                 lambda: bk.FP8KVCache(w.payload_d[:, :, ::2], w.scale_d[:, :, ::2].contiguous()), lambda: bk.FP8KVCache.from_planes([], [])):
        with pytest.raises(RuntimeError):
            make()
    # the C entry points, with a workspace that is missing or too small
    d = w.cache._batch(q, t.repeat(1, 200).contiguous(), l, None)      # sequences that may be long: their parts need space
    need = lib.bikv_fp8_attend_workspace(w.cache._h, d, 4)
    assert need > 0
    for ws, size in ((None, need), (q.data_ptr(), need - 1), (q.data_ptr() + 4, need)):
        assert lib.bikv_fp8_attend(w.cache._h, 1, d, q.data_ptr(), 512, 128, 4, 1, 0.1, k.data_ptr(), 512, 128, None, ws, size, None) == _lib.EINVAL
    wide = struct.pack("=7q2i", t.data_ptr(), 1 << 40, 1 << 40, l.data_ptr(), 0, 2, 2, 0, 0)
    assert lib.bikv_fp8_attend_workspace(w.cache._h, wide, 4) == _lib.ERANGE
    for at, value in ((5, -1), (6, -2), (2, -1), (7, 2), (6, 3), (1, 0), (3, 0), (0, 0)):          # n_seqs, n_rows, max_pages, dtype, rows without starts, table stride, null arrays
        f = list(struct.unpack("=7q2i", d))
        f[at] = value
        for call in (lambda b: lib.bikv_fp8_attend(w.cache._h, 1, b, q.data_ptr(), 512, 128, 4, 1, 0.1, k.data_ptr(), 512, 128, None, q.data_ptr(), need, None),
                     lambda b: lib.bikv_fp8_append(w.cache._h, 1, b, k.data_ptr(), 256, 128, k.data_ptr(), 256, 128, None)):
            assert call(struct.pack("=7q2i", *f)) == _lib.EINVAL, (at, value)


# ---- V scales far apart -------------------------------------------------------------------------
def _weight_oracle(w, q, causal=True, layer=1):
    """(out, lse, tolerance of out, tolerance of lse), float64, for pages of any V scale. A row's weights are p_j vs_j over the keys it sees, W the largest of them. A
    weight is rounded to fp16's 11 bits (2^-12 of itself at most) or, far below W, to 2^-25 of W, and multiplies |byte| <= 448; what one bound or
    the other leaves is doubled, for a weight is a product of rounded factors. z is summed in fp32 (dz), the n products too. The output's own
    rounding is eps / 2, or half its type's smallest step."""
    D, G, P = w.D, w.Hq // w.H, w.P
    val = w.bytes[layer].view(FP8).double()
    out = torch.zeros((w.rows, w.Hq, D), dtype=torch.float64)
    lse = torch.full((w.rows, w.Hq), -math.inf, dtype=torch.float64)
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    info = torch.finfo(w.t)
    for b, (n, new) in enumerate(zip(w.lens, w.news)):
        pages = w.table[b, :-(-n // P)]
        r = slice(int(w.starts[b]), int(w.starts[b]) + new)
        for h in range(w.Hq if n and new else 0):
            k, v = (val[kv, pages][:, :, h // G].reshape(-1, D)[:n] for kv in (0, 1))
            ks, vs = (w.scale[layer, kv][pages][:, h // G].double().repeat_interleave(P)[:n] for kv in (0, 1))
            x = q[r, h].double() / math.sqrt(D)
            z = (x @ k.t()) * ks
            see = torch.arange(n)[None] < (n - new + 1 + torch.arange(new))[:, None] if causal else torch.ones(new, n, dtype=torch.bool)
            dz = (D + 4) * 2.0 ** -24 * torch.where(see, (x.abs() @ k.abs().t()) * ks, torch.zeros_like(z)).amax(1)
            z = torch.where(see, z, torch.full_like(z, -math.inf))
            any_ = see.any(1)
            lse[r, h] = torch.logsumexp(z, 1)
            p = torch.where(see, torch.exp(z - torch.where(any_, lse[r, h], torch.zeros_like(lse[r, h]))[:, None]), torch.zeros_like(z))
            weight = p * vs
            out[r, h] = weight @ v
            A, W = weight @ v.abs(), weight.amax(1, keepdim=True)
            tol[r, h] = (info.eps / 2 * out[r, h].abs() + info.smallest_normal * info.eps / 2
                         + A * (2.0 ** -11 + 2 * dz[:, None] + 2.0 ** -20 + (n + 8) * 2.0 ** -24) + n * 448 * W * 2.0 ** -24)
            ltol[r, h] = dz + 2.0 ** -21 * (1 + torch.where(any_, lse[r, h].abs(), torch.zeros_like(dz))) + (n + 8) * 2.0 ** -24
    return out, lse, tol, ltol


def _check_weights(w, q, causal=True):
    got = w.attend(q, causal=causal)
    w.cache.check()
    out, lse, tol, ltol = _weight_oracle(w, q, causal)
    o, l = got[0].cpu().double(), got[1].cpu().double()
    over = (o - out).abs() - tol
    assert not (over > 0).any(), f"out is off by {float(((o - out).abs() / tol).max())} times what it may be"
    none = lse == -math.inf
    assert torch.equal(l == -math.inf, none) and ((l - lse).abs() <= ltol)[~none].all()


FAR = [
    # lens, new tokens, KV heads, q heads per KV head, head size, tokens of a page
    ([200], [40], 2, 4, 128, 16),                                    # many rows
    ([700, 300], [150, 130], 1, 2, 64, 16), ([300], [290], 1, 1, 128, 1), ([1500], [70], 1, 2, 128, 50),
    ([200], [16], 2, 1, 128, 16),                                    # few: 16 rows
    ([77, 200], [5, 3], 2, 4, 64, 8), ([600] + [40] * 9, [5] * 10, 1, 6, 128, 16),        # and 32
    ([400, 90], [1, 1], 2, 8, 128, 16),                              # one token each: it sees every page
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("wide", [0, 9000])
@pytest.mark.parametrize("apart", [5, 8, 9, 20, 26, 36, 150])
@pytest.mark.parametrize("case", range(len(FAR)))
def test_v_scales_of_later_pages_do_not_reach_earlier_rows(bk, cuda, case, apart, wide, dtype):
    """The pages of a sequence's last tokens have V scales 2^apart larger than the ones before: the rows that see none of them keep all of their bits, and
    the same holds the other way round for the rows that do."""
    lens, news, H, G, D, P = FAR[case]
    if dtype == "fp16" and apart > 36:
        apart = 30                                                   # what lies farther apart is no fp16 number
    w = World(bk, cuda, lens, news, P=P, H=H, D=D, Hq=G * H, dtype=dtype, seed=90 + case, wide=wide)
    for b, (n, new) in enumerate(zip(lens, news)):
        pages = w.table[b, :-(-n // P)]
        late = pages[(n - -(-new // 2)) // P:]                       # the later half of the new tokens, and what shares their first page
        w.scale[1, 1, pages] *= 2.0 ** (-70 if apart > 64 else 10 - apart)
        w.scale[1, 1, late] *= 2.0 ** apart
    w.push()
    _check_weights(w, w.randn(w.Hq, 1.5))
    _check_weights(w, w.randn(w.Hq, 1.5), causal=False)


@pytest.mark.parametrize("dtype,apart", [("bf16", 36), ("fp16", 30)])
@pytest.mark.parametrize("G", [1, 2])
def test_v_scales_of_later_pages_in_the_same_step_of_a_wave(bk, cuda, G, dtype, apart):
    """So many tiles that a head has one wave: it reads the last, far larger page together with pages that every row sees."""
    lens = [90 + i % 9 for i in range(140)]
    w = World(bk, cuda, lens, [16] * 140, H=8, D=64, Hq=8 * G, dtype=dtype, seed=105, wide=0)
    for b, n in enumerate(lens):
        w.scale[1, 1, w.table[b, :-(-n // 16)]] *= 2.0 ** (10 - apart)
        w.scale[1, 1, w.table[b, (n - 1) // 16]] *= 2.0 ** apart
    w.push()
    _check_weights(w, w.randn(w.Hq, 1.5))


@pytest.mark.parametrize("wide", [0, 9000])
@pytest.mark.parametrize("case", range(len(FAR)))
def test_v_scales_of_any_kind(bk, cuda, case, wide):
    """Scales from 2^-90 to 2^70 page by page, zeros and the scale of an empty page among them; rows that hardly attend to the pages of large scale."""
    lens, news, H, G, D, P = FAR[case]
    w = World(bk, cuda, lens, news, P=P, H=H, D=D, Hq=G * H, seed=110 + case, wide=wide)
    e = torch.randint(-90, 70, w.scale[1, 1].shape, generator=w.g).double()
    w.scale[1, 1] = torch.exp2(e).float()
    w.scale[1, 1, ::5] = 0.0
    w.scale[1, 1, 3::5] = 2.0 ** -126
    w.push()
    _check_weights(w, w.randn(w.Hq, 1.5))
    _check_weights(w, w.randn(w.Hq, 6.0), causal=False)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("wide", [0, 9000])
@pytest.mark.parametrize("news,G", [([1], 4), ([16], 1), ([6], 5), ([150], 2)])
def test_a_page_that_a_row_hardly_attends_to_takes_no_bits(bk, cuda, news, G, wide, dtype):
    """Keys of the large V scale lie some 2^-60 below the others in the softmax: the others' values are what comes out."""
    w = World(bk, cuda, [260], news, H=2, Hq=2 * G, dtype=dtype, seed=130, wide=wide)
    w.bytes[1, 0] = 0x38                                             # every key is 1 in every place
    w.scale[1, 0] = 2.0 ** -2
    far = w.table[0, 2:9:3]
    w.scale[1, 0, far] = 2.0 ** -7                                   # z = 16 sqrt(2) there ...
    w.scale[1, 1] = 2.0 ** -20
    w.scale[1, 1, far] = 2.0 ** (9 if dtype == "fp16" else 30)
    w.push()
    q = (1 + torch.rand((w.rows, w.Hq, 128), generator=w.g) * 0.1).to(w.t) * 16
    _check_weights(w, q)
    _check_weights(w, q, causal=False)


def test_calls_of_more_work_than_a_launch_has_threads_for_are_refused(bk, lib, cuda):
    """As what they are, and before anything is launched: the sizes are numbers here, no memory stands behind them."""
    from bikv_pagecopy import _lib
    cache = bk.FP8KVCache(torch.zeros(1, 2, 4, 1, 64, 64, dtype=torch.uint8, device=cuda), torch.ones(1, 2, 4, 64, device=cuda))
    x = torch.zeros(64, 64, 64, dtype=torch.bfloat16, device=cuda)
    table, lens, starts = (torch.zeros(n, dtype=torch.int64, device=cuda) for n in (4, 4, 5))
    at = lambda seqs, rows, pages, starts: struct.pack("=7q2i", table.data_ptr(), pages, pages, lens.data_ptr(), starts, seqs, rows, 0, 0)
    for batch in (at(1, 600000, 4, starts.data_ptr()), at(1 << 20, 1 << 20, 4, 0)):
        assert lib.bikv_fp8_append(cache._h, 0, batch, x.data_ptr(), 4096, 64, x.data_ptr(), 4096, 64, None) == _lib.ERANGE
        assert "too many" in _lib.last_error()
    for batch in (at(5000000, 5000000, 4, 0), at(1 << 20, 1 << 26, 4, starts.data_ptr())):
        assert lib.bikv_fp8_attend_workspace(cache._h, batch, 64) == _lib.ERANGE
        assert lib.bikv_fp8_attend(cache._h, 0, batch, x.data_ptr(), 4096, 64, 64, 1, 0.1, x.data_ptr(), 4096, 64, None, None, 0, None) == _lib.ERANGE
    cache.check()


def test_tensors_with_a_forward_mode_gradient_are_refused(bk, cuda):
    import torch.autograd.forward_ad as fa
    w = World(bk, cuda, [40, 20], [1, 1], H=2, Hq=4, seed=140, ragged=False)
    k, q = w.randn(2).to(cuda), w.randn(4).to(cuda)
    with fa.dual_level():
        dual = lambda x: fa.make_dual(x, torch.ones_like(x))
        for bad in (lambda: w.cache.attend(1, dual(q), w.table_d, w.lens_d), lambda: w.cache.append(1, dual(k), k, w.table_d, w.lens_d),
                    lambda: w.cache.append(1, k, dual(k), w.table_d, w.lens_d), lambda: w.cache.attend(1, q, w.table_d, w.lens_d, out=dual(q.clone()))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                bad()
        w.cache.attend(1, q, w.table_d, w.lens_d)
    w.cache.check()
    assert torch.equal(w.payload_d.cpu().view(torch.uint8), w.bytes)


def test_a_cache_over_tensors_that_want_a_gradient_is_refused(bk, cuda):
    w = World(bk, cuda, [40], [1], H=2, Hq=4, seed=141, ragged=False)
    learnt = w.scale_d.clone().requires_grad_()
    planes = [w.payload_d[l, kv] for l in range(2) for kv in (0, 1)]
    scales = [w.scale_d[l, kv] for l in range(2) for kv in (0, 1)]
    for make in (lambda: bk.FP8KVCache(w.payload_d, learnt), lambda: bk.FP8KVCache.from_planes(planes, scales[:3] + [scales[3].clone().requires_grad_()])):
        with pytest.raises(RuntimeError, match="gradient"):
            make()
        with torch.no_grad():
            make().close()


@pytest.mark.parametrize("wide", [0, 9000])
@pytest.mark.parametrize("news,G", [([20], 1), ([9], 3), ([140], 2)])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_a_scale_that_is_not_finite_among_scales_far_apart(bk, cuda, value, news, G, wide):
    """Rows that do not see its page are what they are without it; the others are not finite."""
    w = World(bk, cuda, [208], news, P=16, H=1, Hq=G, seed=142, wide=wide)
    w.bytes[1][:, int(w.table[0, 12])] |= 0x08                     # no zero among its bytes: 0 * inf would hide nothing
    w.scale[1, 1, w.table[0, 1:13:3]] *= 2.0 ** 40
    w.scale[1, 1, w.table[0, 2]] = 0.0
    w.push()
    q = w.randn(G)
    out, _, tol, _ = _weight_oracle(w, q)
    w.scale_d[1, 1, int(w.table[0, 12])] = value                   # tokens 192 .. 207
    got = w.attend(q)
    w.cache.check()
    o, first = got[0].cpu().double(), 192 - (208 - news[0])
    first = max(first, 0)
    assert ((o[:first] - out[:first]).abs() <= tol[:first]).all() and not o[first:].isfinite().any()


def test_scales_far_apart_give_the_same_bits_and_replay_from_a_graph(bk, cuda):
    for lens, news, G in (([500, 90, 33], [1, 1, 1], 4), ([300, 80], [3, 5], 6), ([700, 300], [200, 140], 2)):
        w = World(bk, cuda, lens, news, H=2, Hq=2 * G, seed=143, wide=9000 * (G == 4))
        w.scale[1, 1] *= torch.exp2(torch.randint(-30, 1, w.scale[1, 1].shape, generator=w.g).float())
        w.push()
        q = w.randn(2 * G).to(cuda)
        want = w.cache.attend(1, q, w.table_d, w.lens_d, w.starts_d, return_lse=True)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out, lse = w.cache.attend(1, q, w.table_d, w.lens_d, w.starts_d, return_lse=True)
        for _ in range(3):
            out.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
        _check_weights(w, q.cpu())
