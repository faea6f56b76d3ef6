"""Log probabilities of given tokens, entropies and top alternatives against plain torch in 64 bits."""
import math

import pytest
import torch

from b200serve.ops import logprob as LP

gpu = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")
LOWEST = torch.finfo(torch.float32).min
U = 2.0 ** -24           # half a step of fp32, relative


def reference(z, tokens, top):
    """The definition in 64 bits: log probability, entropy, ids and log probabilities of the alternatives."""
    z = z.double()
    m, n = z.shape
    lp = torch.log_softmax(z, dim=1)
    none = (z == -INF).all(1)
    lp[none] = -INF
    p = lp.exp()
    h = -torch.where(p > 0, p * lp, 0.0).sum(1)
    h[torch.isnan(lp).any(1)] = NAN
    t = tokens.long()
    inside = (t >= 0) & (t < n)
    got = torch.where(inside, lp.gather(1, t.clamp(0, n - 1)[:, None])[:, 0], NAN)
    order = torch.where(torch.isnan(z), -INF, z)
    ids = order.sort(dim=1, descending=True, stable=True).indices
    if torch.isnan(z).any():                      # NaN last, behind -inf
        rank = torch.where(torch.isnan(z), 2.0, torch.where(z == -INF, 1.0, 0.0))
        ids = ids.gather(1, rank.gather(1, ids).sort(dim=1, stable=True).indices)
    ids = ids[:, :top]
    top_lp = lp.gather(1, ids)
    pad = top - ids.shape[1]
    if pad:
        ids = torch.cat([ids, ids.new_full((m, pad), -1)], 1)
        top_lp = torch.cat([top_lp, top_lp.new_full((m, pad), -INF)], 1)
    return got, h, ids.int(), top_lp


def bounds(z, dz=0.0):
    """What fp32 may add up to, per row: (of ln S, of the entropy), and a factor of |z - max| for a single log probability.

    A term exp d of S is off by: d rounded (|d| U), d times log2 e rounded and log2 e itself (2 |d| U together), ex2.approx (4 U); a sum
    of at most 256 additions on its way adds 256 U.  So S is off by (260 + 3 E|d|) U relative, with E|d| = sum p |d| = ln S - H, and
    ln S, at most 20 here, by that and one rounding of itself (log1pf: 2 U).  H = ln S + E|d|: each term d exp d is off by another
    U |d|, and d itself counts in E d^2, at most 200 E|d|; its terms that are not negligible have |d| < 20.  ``dz``: error of a logit."""
    z = z.double()
    d = z - z.max(1, keepdim=True).values
    p = torch.softmax(z, 1)
    mean = torch.where(p > 0, p * -d, 0.0).sum(1)
    square = torch.where(p > 0, p * d * d, 0.0).sum(1)
    rel = (260 + 3 * mean) * U
    lse = rel + 2 * 20 * U + 2 * dz
    return lse, lse + (262 * mean + 4 * square) * U + rel * mean + 2 * dz * (1 + mean)


def close(got, want, tol):
    """Equal where not finite, else within ``tol`` (per element)."""
    got, want = got.double(), want.double()
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[~fin & ~torch.isnan(want)], want[~fin & ~torch.isnan(want)])
    err = (got - want).abs()[fin]
    tol = torch.as_tensor(tol, device=got.device).expand_as(want)[fin]
    assert bool((err <= tol).all()), (float((err - tol).max()), float(err.max()))


def check(out, z, tokens, top, dz=0.0, ids=True):
    lp, h, want_ids, top_lp = reference(z, tokens, top)
    lse, ent = bounds(z, dz)
    close(out.logprob, lp, lse.nan_to_num(0.0) + lp.abs().nan_to_num(0.0, 0.0, 0.0) * 2 * U)
    close(out.entropy, h, ent.nan_to_num(0.0) + h.abs().nan_to_num(0.0) * 2 * U)
    if ids:
        assert torch.equal(out.top_ids, want_ids)
    close(out.top_logprobs, top_lp, lse.nan_to_num(0.0)[:, None] + top_lp.abs().nan_to_num(0.0, 0.0, 0.0) * 2 * U)


def rand_logits(m, n, seed, ld=None, offset=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    buf = torch.full((m, (ld or n) + offset), NAN, device="cuda")
    z = buf[:, offset: offset + n]
    z.copy_(2.5 * torch.randn(m, n, device="cuda", generator=g))
    z[torch.arange(m), torch.randint(0, n, (m,), device="cuda", generator=g)] += 16 * torch.rand(m, device="cuda", generator=g)
    return z, torch.randint(0, n, (m,), device="cuda", generator=g, dtype=torch.int32)


# ------------------------------------------------------------------ refusals (no GPU needed)
def test_refusals():
    z, t = torch.zeros(2, 8), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        LP.token_logprobs(z, t)
    with pytest.raises(ValueError, match="CUDA"):
        LP.score(torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(8, 64, dtype=torch.bfloat16), t)
    with pytest.raises(ValueError, match="CUDA"):
        LP.score_i8(torch.zeros(2, 64, dtype=torch.bfloat16), (torch.zeros(8, 64, dtype=torch.int8), torch.ones(8)), t)
    for top in (LP.MAX_TOP + 1, -1):
        with pytest.raises(ValueError, match="at most"):
            LP.Logprobs.empty(2, top, "cpu")
    out = LP.Logprobs.empty(2, 4, "cpu")
    for m, top in ((2, 3), (3, 4), (3, None)):
        with pytest.raises(ValueError, match="asked"):
            LP._results(m, top, out, z.device)
    f = torch.zeros(2, 4)
    for wrong in ((out.logprob[:1], out.entropy, out.top_ids, f), (out.logprob, out.entropy.double(), out.top_ids, f), (out.logprob, out.entropy, out.top_ids.long(), f),
                  (out.logprob, out.entropy, out.top_ids, f[:, :3]), (out.logprob, out.entropy, out.top_ids, torch.zeros(4, 2).T),
                  (out.logprob, out.entropy, torch.zeros(2, 33, dtype=torch.int32), torch.zeros(2, 33))):
        with pytest.raises(ValueError, match="contiguous|at most"):
            LP.Logprobs(*wrong)
    for bad in (t.long(), t[:1], torch.zeros(4, dtype=torch.int32)[::2], torch.zeros(2)):
        with pytest.raises(ValueError, match="int32"):
            LP._check_tokens(bad, 2, z.device)


def test_results_of_rows():
    out = LP.Logprobs.empty(5, 3, "cpu")
    part = out.rows(1, 4)
    assert part.logprob.data_ptr() == out.logprob[1:].data_ptr() and part.top_ids.shape == (3, 3) and part.top_logprobs.is_contiguous()


@gpu
def test_refusals_of_shapes_and_strides():
    z, t = torch.zeros(2, 64, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    x, w = (torch.zeros(r, 64, dtype=torch.bfloat16, device="cuda") for r in (2, 8))
    w8, ws = torch.zeros(8, 128, dtype=torch.int8, device="cuda"), torch.ones(8, device="cuda")
    for call in (lambda: LP.token_logprobs(z.bfloat16(), t), lambda: LP.token_logprobs(z.T, t), lambda: LP.token_logprobs(z[0], t),
                 lambda: LP.token_logprobs(z[:, :0], t), lambda: LP.token_logprobs(z[:1].expand(2, 64), t),
                 lambda: LP.token_logprobs(z, t, top=33), lambda: LP.token_logprobs(z, t.cpu()),
                 lambda: LP.score(x.float(), w, t), lambda: LP.score(x, w.float(), t), lambda: LP.score(x[:, :56], w, t), lambda: LP.score(x, w[:0], t),
                 lambda: LP.score(x[:, :40], w[:, :40], t), lambda: LP.score(torch.zeros(2, 68, dtype=torch.bfloat16, device="cuda"), w, t),
                 lambda: LP.score(torch.zeros(2, 72, dtype=torch.bfloat16, device="cuda")[:, 1:65], w, t), lambda: LP.score(x, w, t, out=LP.Logprobs.empty(3, 0, "cuda")),
                 lambda: LP.score_i8(x, (w8, ws), t), lambda: LP.score_i8(torch.zeros(2, 128, dtype=torch.bfloat16, device="cuda"), (w8, ws[:3]), t),
                 lambda: LP.score_i8(torch.zeros(2, 128, dtype=torch.bfloat16, device="cuda"), (w8, ws.half()), t),
                 lambda: LP.score_i8(torch.zeros(2, 128, dtype=torch.bfloat16, device="cuda"), (w8.float(), ws), t),
                 lambda: LP.score_i8(torch.zeros(2, LP.MAX_I8_COLUMNS + 16, dtype=torch.bfloat16, device="cuda"),
                                     (torch.zeros(8, LP.MAX_I8_COLUMNS + 16, dtype=torch.int8, device="cuda"), ws), t)):
        with pytest.raises(ValueError):
            call()


# ------------------------------------------------------------------ rows of logits
@gpu
@pytest.mark.parametrize("n", [1, 2, 31, 33, 700, 1023, 1025, 4096, 8193, 33000, 102397, 151936, 262147, 600001])
@pytest.mark.parametrize("m,top", [(1, 0), (1, 5), (3, 20), (2, 32)])
def test_rows(m, n, top):
    z, t = rand_logits(m, n, 31 * m + n)
    check(LP.token_logprobs(z, t, top), z, t, top)


@gpu
@pytest.mark.parametrize("m", [8, 64, 150, 500, 1200])
@pytest.mark.parametrize("n,top", [(1000, 3), (16385, 20), (40001, 0)])
def test_many_rows(m, n, top):
    z, t = rand_logits(m, n, m + n)
    check(LP.token_logprobs(z, t, top), z, t, top)


@gpu
@pytest.mark.parametrize("ld,offset", [(5000, 0), (5001, 0), (5002, 1), (5003, 3), (5000, 2)])
def test_rows_of_wider_buffers(ld, offset):
    """Columns beside the vocabulary hold NaN: none is read."""
    for m in (1, 5, 300):
        z, t = rand_logits(m, 4999, m, ld, offset)
        check(LP.token_logprobs(z, t, 7), z, t, 7)


@gpu
def test_rows_that_leave_nothing():
    n, top = 5003, 8
    z = torch.randn(16, n, device="cuda")
    t = torch.full((16,), 11, dtype=torch.int32, device="cuda")
    z[0] = -INF                                   # every id banned
    z[1] = -INF; z[1, 4321] = 2.0                 # one left, the token among the banned
    z[2] = -INF; z[2, 11] = -3e38                 # the token alone is left
    z[3] = LOWEST                                 # masked by the lowest number: all alike
    z[4, 1:] = LOWEST                             # and one above it
    z[5, 17] = NAN
    z[6, 4000] = INF
    z[7] = NAN
    z[8, 100:] = -INF                             # NaN beside banned ids
    z[8, 3] = NAN
    z[9] = -INF; z[9, 5] = NAN
    z[10] = 0.0; z[10, 1::2] = -0.0               # one value: ties by id
    z[11] = 3.0                                   # all equal
    z[12, 11] = 3e38                              # spread beyond fp32
    z[12, 12] = -3e38
    z[13] = INF
    t[14], t[15] = -1, n
    check(LP.token_logprobs(z, t, top), z, t, top)
    wide = torch.full((6, 200000), -INF, device="cuda")
    wide[1, 199999], wide[2, 77777] = 1.0, NAN
    wide[3] = NAN                                 # no number at all; three banned ids far in; numbers, a banned id and the rest NaN
    wide[4] = NAN; wide[4, [1000, 1001, 199990]] = -INF
    wide[5] = NAN; wide[5, 150000:150004] = 1.0; wide[5, 7] = -INF
    tw = torch.tensor([5, 199999, 3, 0, 1000, 7], dtype=torch.int32, device="cuda")
    check(LP.token_logprobs(wide, tw, 32), wide, tw, 32)


@gpu
@pytest.mark.parametrize("kind", ["ascending", "descending", "ties", "last", "first", "two"])
def test_orders(kind):
    """Orders in which a running selection has most to do, and values that tie across any cut of the row."""
    m, n, top = 4, 151936, 32
    i = torch.arange(n, device="cuda", dtype=torch.float32)
    g = torch.Generator(device="cuda").manual_seed(5)
    z = {"ascending": i / n * 20, "descending": (n - i) / n * 20, "ties": (i % 7) / 2, "last": (i >= n - 40) * 9.0, "first": (i < 40) * 9.0,
         "two": torch.where(torch.rand(n, device="cuda", generator=g) < 0.5, 1.0, 1.5)}[kind].expand(m, n).contiguous()
    t = torch.tensor([0, 1, n // 2, n - 1], dtype=torch.int32, device="cuda")
    check(LP.token_logprobs(z, t, top), z, t, top)


@gpu
@pytest.mark.parametrize("n", [50, 5000, 151936])
def test_sure_tokens_keep_their_digits(n):
    """ln S near zero: S' = (n - 1) exp(-gap) is off by (260 + 3 gap) U relative and log1p adds 2 U, so the log probability of the likely
    token is off by no more, relative; the entropy S' (1 + gap) likewise, and by its rounding."""
    for gap in (15.0, 25.0, 40.0, 80.0):
        z = torch.full((2, n), -gap, device="cuda")
        z[0, 3], z[1, n - 1] = 0.0, 0.0
        t = torch.tensor([3, n - 1], dtype=torch.int32, device="cuda")
        out = LP.token_logprobs(z, t, 1)
        rest = (n - 1) * math.exp(-gap)
        lse = math.log1p(rest)
        tol = (266 + 3 * gap) * U
        assert (out.logprob.double() / -lse - 1).abs().max() <= tol
        assert (out.entropy.double() / (lse + rest * gap / (1 + rest)) - 1).abs().max() <= 2 * tol
        assert out.top_ids[:, 0].tolist() == [3, n - 1]


@gpu
def test_no_rows():
    out = LP.token_logprobs(torch.zeros(0, 100, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda"), 4)
    assert out.top_ids.shape == (0, 4)


@gpu
def test_rows_in_a_graph_and_on_streams():
    z, t = rand_logits(6, 151936, 3)
    want = LP.token_logprobs(z, t, 9)
    out = LP.Logprobs.empty(6, 9, "cuda")
    LP.token_logprobs(z, t, out=out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        LP.token_logprobs(z, t, out=out)
    z2, t2 = rand_logits(6, 151936, 4)
    want2 = LP.token_logprobs(z2, t2, 9)
    z.copy_(z2)
    t.copy_(t2)
    g.replay()
    for a, b in zip(vars(out).values(), vars(want2).values()):
        assert torch.equal(a, b)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    z3, t3 = rand_logits(6, 151936, 3)
    torch.cuda.synchronize()
    with torch.cuda.stream(a):
        o1 = LP.token_logprobs(z3, t3, 9)
    with torch.cuda.stream(b):
        o2 = LP.token_logprobs(z2, t2, 9)
    torch.cuda.synchronize()
    for o, w in ((o1, want), (o2, want2)):
        assert all(torch.equal(x, y) for x, y in zip(vars(o).values(), vars(w).values()))


# ------------------------------------------------------------------ rows through the head
def grid(shape, seed, steps, scale):
    """bf16 values on a coarse grid around zero: products and sums of a few thousand of them are whole numbers of steps below 2^24, so an
    fp32 sum in any order is exact."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * steps).round_().clamp_(-127, 127).mul_(scale).bfloat16()


@gpu
@pytest.mark.parametrize("m", [1, 3, 127, 128, 129, 256, 257, 512, 513, 700])
@pytest.mark.parametrize("n,k,top", [(1, 64, 0), (5, 72, 8), (255, 64, 0), (257, 200, 3), (1000, 512, 0), (2051, 136, 32), (20000, 384, 0)])
def test_score(m, n, k, top):
    x, w = grid((m, k), m + n, 12, 1 / 16), grid((n, k), m + n + 1, 20, 1 / 64)
    t = torch.randint(0, n, (m,), device="cuda", dtype=torch.int32)
    t[0] = n - 1
    if m > 2:
        t[1], t[2] = -1, n
    check(LP.score(x, w, t, top), x.double() @ w.double().T, t, top)


@gpu
@pytest.mark.parametrize("m", [1, 100, 130, 300, 600])
@pytest.mark.parametrize("n,k,top", [(3, 128, 2), (257, 200, 0), (1000, 512, 5), (20003, 144, 0)])
def test_score_i8(m, n, k, top):
    g = torch.Generator(device="cuda").manual_seed(m + n)
    x = torch.randn(m, k, device="cuda", generator=g).bfloat16()
    pad = (k + 15) // 16 * 16
    w8 = torch.randint(-127, 128, (n, pad), device="cuda", generator=g, dtype=torch.int8)[:, :k]
    ws = (0.5 + torch.rand(n, device="cuda", generator=g)) / 300
    t = torch.randint(0, n, (m,), device="cuda", dtype=torch.int32)
    t[0] = n - 1
    xf = x.float()
    largest = xf.abs().amax(1, keepdim=True)
    s = largest / torch.full_like(largest, 127)            # (a division by a number is a product with its rounded inverse on the GPU)
    acc = (xf * (1 / s)).round().double() @ w8.double().T
    # the sum as fp32 and two products, rounded one by one, are the logits: their ids are the ones
    z = (acc.float() * s) * ws
    check(LP.score_i8(x, (w8, ws), t, top), z, t, top)
    if top:      # in 64 bits: three roundings of a logit
        exact = acc * s.double() * ws.double()
        check(LP.score_i8(x, (w8, ws), t, top), exact, t, top, dz=float(exact.abs().max()) * 3 * U, ids=False)


@gpu
@pytest.mark.parametrize("m,n,k", [(200, 5000, 2048), (70, 3001, 5120)])
def test_score_of_values_that_round(m, n, k):
    """Arbitrary values: a logit is a sum of k products in fp32, each addition (at most k of them) off by a step, 2 U, of what has been
    summed so far, which no partial sum of |x w| exceeds."""
    g = torch.Generator(device="cuda").manual_seed(k)
    x, w = torch.randn(m, k, device="cuda", generator=g).bfloat16(), (0.03 * torch.randn(n, k, device="cuda", generator=g)).bfloat16()
    t = torch.randint(0, n, (m,), device="cuda", dtype=torch.int32)
    # additions of tensor cores: groups of 16 products and one addition to the accumulator each
    dz = float((x.double().abs() @ w.double().abs().T).max()) * 2 * U * (k / 16 + 16)
    z = x.double() @ w.double().T
    for top in (0, 6):
        check(LP.score(x, w, t, top), z, t, top, dz=dz, ids=False)


@gpu
def test_score_of_strided_rows():
    buf, head = grid((90, 256), 1, 12, 1 / 16), grid((600, 320), 2, 20, 1 / 64)
    x, w = buf[:, 64:200], head[:, 8:144]
    t = torch.randint(0, 600, (90,), device="cuda", dtype=torch.int32)
    for top in (0, 4):
        check(LP.score(x, w, t, top), x.double() @ w.double().T, t, top)
    check(LP.score(x[::2], w, t[::2].contiguous(), 2), x[::2].double() @ w.double().T, t[::2], 2)
    check(LP.score(x[5:6], w[7:8], torch.zeros_like(t[:1])), x[5:6].double() @ w[7:8].double().T, torch.zeros_like(t[:1]), 0)


@gpu
@pytest.mark.parametrize("top", [0, 5])
def test_score_in_slabs(monkeypatch, top):
    """More rows than the logits that are kept at a time."""
    monkeypatch.setattr(LP, "SLAB_ELEMS", 256 * 1000)
    x, w = grid((600, 128), 3, 12, 1 / 16), grid((999, 128), 4, 20, 1 / 64)
    t = torch.randint(0, 999, (600,), device="cuda", dtype=torch.int32)
    check(LP.score(x, w, t, top), x.double() @ w.double().T, t, top)


@gpu
@pytest.mark.parametrize("top", [0, 3])
def test_score_of_rows_and_heads_without_numbers(top):
    """NaN and infinities of a row or of the head stay with the rows that they meet."""
    n, k, m = 700, 128, 300
    x, w = grid((m, k), 5, 12, 1 / 16), grid((n, k), 6, 20, 1 / 64)
    t = torch.randint(0, n, (m,), device="cuda", dtype=torch.int32)
    x[4, 7], x[130, 0], x[299, 127] = NAN, INF, -INF
    x[6] = 0                                                    # all logits 0
    z = x.double() @ w.double().T
    got = LP.score(x, w, t, top)
    bad = torch.zeros(m, dtype=torch.bool, device="cuda")
    bad[[4, 130, 299]] = True
    assert bool(torch.isnan(got.logprob[bad]).all()) and bool(torch.isnan(got.entropy[bad]).all())
    keep = ~bad
    check(LP.Logprobs(*(v[keep] for v in vars(got).values())), z[keep], t[keep], top)
    w8, ws = (w * 64).to(torch.int8), torch.full((n,), 1 / 64, device="cuda")
    got = LP.score_i8(x, (w8, ws), t, top)
    assert bool(torch.isnan(got.logprob[bad]).all()) and bool(torch.isfinite(got.logprob[keep]).all())
    close(got.entropy[6:7], torch.tensor([math.log(n)], device="cuda"), 300 * U)
    tiny = torch.full((2, k), 2.0 ** -133, dtype=torch.bfloat16, device="cuda")      # the smallest bf16: a scale without an inverse in fp32
    out = LP.score_i8(tiny, (w8, ws), t[:2].contiguous(), top)
    close(out.entropy, torch.full((2,), math.log(n), device="cuda"), 300 * U)


@gpu
@pytest.mark.parametrize("n", [3000, 40000])
def test_score_of_ties(n):
    """Rows whose logits are all alike, or of two values: more chunks reach the bound than are noted."""
    x, w = grid((5, 128), 21, 12, 1 / 16), torch.zeros(n, 128, dtype=torch.bfloat16, device="cuda")
    w[:, 0] = (torch.arange(n, device="cuda") % 3 == 1).bfloat16()
    x[:, 0] = torch.tensor([1.0, 0.0, -1.0, 2.0, -0.5], device="cuda")
    t = torch.tensor([0, 1, 2, n - 1, -1], dtype=torch.int32, device="cuda")
    for top in (1, 32):
        check(LP.score(x, w, t, top), x.double() @ w.double().T, t, top)


@gpu
def test_score_of_ragged_columns():
    """Rows of columns that no 16 bytes hold: a matrix cut out of a wider one."""
    for k in (129, 135, 200, 257):
        x, w = grid((70, 272), 22, 12, 1 / 16)[:, :k], grid((900, 272), 23, 20, 1 / 64)[:, :k]
        t = torch.randint(0, 900, (70,), device="cuda", dtype=torch.int32)
        check(LP.score(x, w, t, 3), x.double() @ w.double().T, t, 3)
        w8, ws = (w * 64).to(torch.int8), torch.full((900,), 1 / 64, device="cuda")
        w8 = torch.nn.functional.pad(w8, (0, 272 - k), value=3)[:, :k]      # beside the columns: something that must not count
        largest = x.float().abs().amax(1, keepdim=True)
        s = largest / torch.full_like(largest, 127)
        z = ((x.float() * (1 / s)).round().double() @ w8.double().T).float() * s * ws
        check(LP.score_i8(x, (w8, ws), t, 3), z, t, 3)


@gpu
def test_score_with_little_room(monkeypatch):
    """No room for the logits of all rows: fewer at a time."""
    x, w = grid((700, 128), 24, 12, 1 / 16), grid((999, 128), 25, 20, 1 / 64)
    t = torch.randint(0, 999, (700,), device="cuda", dtype=torch.int32)
    want, sizes, real = LP.score(x, w, t, 4), [], torch.empty

    def empty(*a, **kw):
        if a and isinstance(a[0], int) and a[0] > 400 * 1000:
            sizes.append(a[0])
            raise torch.OutOfMemoryError("no room")
        return real(*a, **kw)
    out = LP.Logprobs.empty(700, 4, "cuda")
    monkeypatch.setattr(torch, "empty", empty)
    LP.score(x, w, t, out=out)
    monkeypatch.undo()
    assert len(sizes) >= 1
    for a, b in zip(vars(out).values(), vars(want).values()):
        assert torch.equal(a, b) or float((a - b).abs().max()) <= 1e-5


@gpu
def test_score_in_a_graph():
    x, w = grid((300, 256), 7, 12, 1 / 16), grid((5000, 256), 8, 20, 1 / 64)
    t = torch.randint(0, 5000, (300,), device="cuda", dtype=torch.int32)
    for top in (0, 4):
        out = LP.Logprobs.empty(300, top, "cuda")
        LP.score(x, w, t, out=out)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            LP.score(x, w, t, out=out)
        keep = x.clone()
        x.copy_(grid((300, 256), 9, 12, 1 / 16))
        g.replay()
        check(out, x.double() @ w.double().T, t, top)
        x.copy_(keep)


@gpu
def test_scores_at_once():
    """Two products on two streams share nothing."""
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    w = grid((9000, 512), 10, 20, 1 / 64)
    xs = [grid((700, 512), 11 + i, 12, 1 / 16) for i in range(2)]
    t = torch.randint(0, 9000, (700,), device="cuda", dtype=torch.int32)
    want = [LP.score(x, w, t) for x in xs]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for st, x in zip((a, b), xs):
            with torch.cuda.stream(st):
                got.append(LP.score(x, w, t))
        torch.cuda.synchronize()
        for o, v in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(vars(o).values(), vars(v).values()))
