"""Scores through heads of real width: accumulators and scale buffers that are used again and again by a CTA, and products in several pieces."""
import pytest
import torch

from b200serve.ops import lib as K
from b200serve.ops import logprob as LP
from test_logprob import check, grid

pytestmark = pytest.mark.gpu


def i8_case(m, n, k, seed):
    """(x, head, logits): int8 sums are whole numbers, and two products in fp32 follow, rounded one by one."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(m, k, device="cuda", generator=g).bfloat16()
    w8 = torch.randint(-127, 128, (n, k), device="cuda", generator=g, dtype=torch.int8)
    ws = (0.5 + torch.rand(n, device="cuda", generator=g)) / 300
    xf = x.float()
    largest = xf.abs().amax(1, keepdim=True)
    s = largest / torch.full_like(largest, 127)
    # (whole sums below 128 x 127 x 127 < 2^24: exact in fp32 whatever their order)
    acc = (xf * (1 / s)).round().double() @ w8.double().T
    return x, (w8, ws), (acc.float() * s) * ws


def tokens_of(m, n, seed):
    t = torch.randint(0, n, (m,), generator=torch.Generator().manual_seed(seed)).int()
    t[0] = n - 1
    if m > 3:
        t[1], t[2], t[3] = -1, n, 0
    return t.cuda()


# With 148 SMs: 1 row 5 tiles a CTA, 77 and 128 rows 3 to 5, 300 and 384 rows 9 to 13; pairs (129, 256, 385, 512 rows) 6 to 17; 600 rows in turn.
@pytest.mark.parametrize("m", [1, 77, 128, 129, 256, 300, 384, 385, 512, 600])
@pytest.mark.parametrize("n", [102397, 151936])
@pytest.mark.parametrize("k,top", [(64, 0), (64, 5), (128, 20)])
def test_score_goes_on_through_a_range(m, n, k, top):
    """Few columns of k: the sums are what the multiplication waits for, so that an accumulator's reuse is waited for."""
    x, w, t = grid((m, k), m + n, 12, 1 / 16), grid((n, k), m + n + 1, 20, 1 / 64), tokens_of(m, n, m)
    check(LP.score(x, w, t, top), x.double() @ w.double().T, t, top)


@pytest.mark.parametrize("m", [1, 77, 128, 129, 256, 300, 384, 512, 600])
@pytest.mark.parametrize("n", [102397, 151936])
@pytest.mark.parametrize("top", [0, 5])
def test_score_i8_goes_on_through_a_range(m, n, top):
    x, head, z = i8_case(m, n, 128, m + n)
    t = tokens_of(m, n, m + 1)
    check(LP.score_i8(x, head, t, top), z, t, top)


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("m,top", [(600, 0), (600, 5), (513, 0), (900, 3), (512, 0)])
def test_score_in_pieces(monkeypatch, kind, m, top):
    """More rows than are taken at a time, with and without alternatives: pieces of another form than the whole, a last one of another size."""
    n, k = 5003, 128
    if kind == "bf16":
        x, head = grid((m, k), 3, 12, 1 / 16), grid((n, k), 4, 20, 1 / 64)
        z, call = x.double() @ head.double().T, LP.score
    else:
        x, head, z = i8_case(m, n, k, 5)
        call = LP.score_i8
    t = tokens_of(m, n, 6)
    n0 = K.launch_count
    check(call(x, head, t, top), z, t, top)
    one = K.launch_count - n0
    monkeypatch.setattr(LP, "SLAB_ELEMS", 256 * n)
    monkeypatch.setattr(LP, "SLAB_ROWS", 256)
    n0 = K.launch_count
    check(call(x, head, t, top), z, t, top)
    assert K.launch_count - n0 == one * ((m + 255) // 256)
    out = LP.Logprobs.empty(m, top, "cuda")
    out.logprob.fill_(7.0)
    call(x[256:], head, t[256:], out=out.rows(256, m))      # the rows before are left as they were
    assert bool((out.logprob[:256] == 7.0).all())
    check(out.rows(256, m), z[256:], t[256:], top)
