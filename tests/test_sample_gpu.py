"""fml_sample against a plain implementation in Python floats (tokens equal, probabilities to 1e-6).

A weight is a whole multiple of 2^-44 of the largest, so a sum of n weights is off by at most n 2^-45 (n = 2^18: 7.5e-9); a draw or a
cut that lies nearer to the next outcome than 4 n 2^-44 may go either way and is not compared (`near`).  Probabilities: one rounding to
fp32 and the sum's 7.5e-9.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from fluidml_b200 import cabi
from serving_oracle import TYPES, sample as oracle

INF = math.inf


def check(logits, u, temperature=None, top_k=None, top_p=None, min_p=None, tokens_type=torch.int64):
    n, v = logits.shape
    dev = lambda x, t=torch.float32: None if x is None else torch.tensor(x, dtype=t).cuda() if not torch.is_tensor(x) else x.cuda()  # noqa: E731
    tokens, prob = torch.full((n,), -7, dtype=tokens_type).cuda(), torch.full((n,), -7.0).cuda()
    args = dict(temperature=dev(temperature), top_k=dev(top_k, torch.int32), top_p=dev(top_p), min_p=dev(min_p))
    u = torch.as_tensor(u, dtype=torch.float32)
    cabi.sample(logits.cuda(), u.cuda(), tokens, probabilities=prob, **args)
    torch.cuda.synchronize()
    compared = 0
    off = {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0}
    for r in range(n):
        row = [off[k] if a is None else a[r].item() for k, a in args.items()]
        token, p, near = oracle(logits[r].float().tolist(), u[r].item(), *row)
        # an equal distance of zero is a tie by construction (equal weights), which both sides decide alike
        if 0 < near < 4 * v * 2.0 ** -44:
            continue
        compared += 1
        assert tokens[r].item() == token, (r, row, u[r].item(), tokens[r].item(), token)
        assert prob[r].item() == pytest.approx(p, rel=1e-6, abs=1e-30)
    assert compared >= n - 1


def randn(seed, *shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


def rand(seed, n):
    return torch.rand(n, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 4096, 5001, 20011])
def test_no_filter_and_every_filter(dtype, vocab):
    n = 6
    z = (randn(vocab, n, vocab) * 3).to(TYPES[dtype])
    u = rand(1, n)
    check(z, u)
    check(z, u, temperature=[0.3, 1.0, 2.5, 0.0, -1.0, 0.8])
    check(z, u, top_k=[1, 2, 40, vocab, 0, vocab // 2])
    check(z, u, top_p=[0.01, 0.3, 0.9, 0.999, 1.0, 0.0])
    check(z, u, min_p=[0.001, 0.02, 0.2, 1.0, 0.0, 2.0])
    check(z, u, temperature=[0.7, 1.3, 1.0, 0.5, 2.0, 0.9], top_k=[50, 700, 3, 0, 200, 17], top_p=[0.9, 0.95, 0.5, 0.8, 0.99, 0.2],
          min_p=[0.0, 0.01, 0.1, 0.05, 0.001, 0.3], tokens_type=torch.int32)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_ties_go_to_the_lowest_index(dtype):
    z = torch.zeros(9, 3001, dtype=TYPES[dtype])
    z[1:3, 1500:] = 1.0
    z[3, ::7] = 2.0
    z[4] = -0.0
    z[4, ::2] = 0.0  # both zeros are one
    u = rand(3, 9)
    u[0], u[4] = 0.5, 0.25
    check(z, u)
    check(z, u, top_k=[5, 10, 1502, 429, 100, 3000, 2999, 1, 1500])
    check(z, u, top_p=[0.5, 0.25, 0.9, 0.125, 0.5, 0.0, 0.999, 0.75, 0.3])
    check(z, u, top_k=[100, 1600, 20, 500, 64, 64, 64, 64, 64], top_p=[0.5, 0.99, 0.5, 0.5, 0.5, 0.25, 0.125, 1.0, 0.75])
    check(z, u, temperature=[0.0] * 9)


def test_rows_that_leave_little():
    z = randn(5, 8, 777)
    z[0] = -INF
    z[1] = math.nan
    z[2] = -INF
    z[2, 400] = -3.0e38
    z[3, ::2] = INF
    z[4] = torch.finfo(torch.float32).min
    z[4, 5:9] = 1.0
    z[5, ::3] = math.nan
    z[6] = 3.0e38
    z[6, 100] = -3.0e38
    z[7] = torch.finfo(torch.float32).min  # every token masked by the lowest number: all alike
    u = rand(6, 8)
    check(z, u)
    check(z, u, temperature=[0.0] * 8)
    check(z, u, temperature=[INF, INF, INF, 1.0, 3.0, 1e-38, INF, 1e30])
    check(z, u, top_k=[3] * 8, top_p=[0.6] * 8, min_p=[0.05] * 8)
    check(z, u, top_k=[600] * 8, top_p=[0.95] * 8)


def test_uniforms_at_their_ends():
    z = randn(7, 6, 900)
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, -1.0, math.nan, 2.0 ** -24])
    check(z, u)
    z[:, :50] = -INF
    z[:, 850:] = -INF
    check(z, u)
    check(z, u, top_p=[0.9] * 6)


def test_parameters_that_mean_off():
    z, u = randn(8, 4, 500), rand(9, 4)
    check(z, u, top_k=[-3, 0, 500, 10 ** 9], top_p=[1.0, 2.0, math.nan, 1.5], min_p=[0.0, -1.0, math.nan, 0.0])


def test_cold_and_hot_rows():
    z, u = randn(10, 6, 6000) * 4, rand(11, 6)
    check(z, u, temperature=[1e-3, 0.05, 10.0, 100.0, 1e4, 1e-30], top_p=[0.9] * 6)
    check(z, u, temperature=[1e-3, 0.05, 10.0, 100.0, 1e4, 0.2], top_k=[3000] * 6, top_p=[0.7] * 6, min_p=[0.01] * 6)
    check(z * 1e-3 + 100.0, u, top_p=[0.5] * 6, top_k=[0, 0, 1000, 4000, 0, 1])  # neighbours in the last bits
    check(z * 1e-30, u, top_p=[0.5] * 6, top_k=[0, 0, 1000, 4000, 0, 1])


@pytest.mark.parametrize("dtype,vocab", [("f32", 4201), ("f16", 8201), ("bf16", 8201)])
def test_cuts_in_ranges_of_many_keys(dtype, vocab):
    """The cut's bin holds more keys than a histogram has bins, so that the CTAs of a row narrow it in several rounds: fp32 always, 16-bit
    types around zero, where a bin has all the small numbers.  Every CTA has to see the same sums in every round, run after run."""
    n = 4
    z, u = (randn(21, n, vocab) * 1.5).to(TYPES[dtype]), rand(22, n)
    w = torch.exp(z.double())
    top_p = ((w * (z > 0)).sum(1) / w.sum(1)).float()  # the cut falls on the first number that is not above zero, or next to it
    top_k = torch.tensor([0, vocab - 1, vocab // 2 + 2000, 0], dtype=torch.int32)
    check(z, u, top_p=top_p)
    check(z, u, top_p=top_p, top_k=top_k, min_p=[0.0, 1e-4] * 2)
    z, u, top_p, top_k = z.cuda().repeat(64, 1), u.cuda().repeat(64), top_p.cuda().repeat(64), top_k.cuda().repeat(64)
    first = None
    for _ in range(100):
        tokens = torch.empty(64 * n, dtype=torch.int64).cuda()
        cabi.sample(z, u, tokens, top_p=top_p, top_k=top_k)
        first = tokens if first is None else first
        assert torch.equal(tokens.view(64, n), first[:n].expand(64, n))


@pytest.mark.parametrize("dtype,grain", [("f32", 1024), ("bf16", 2048)])
@pytest.mark.parametrize("ctas", [2, 4, 8])
def test_the_largest_logit_from_the_cta_that_has_least_to_do(dtype, grain, ctas):
    """One token more than half as many CTAs take: the last ones have next to nothing to load and are the first to tell the others what
    they found."""
    n, v = 1200, grain * (ctas // 2) + 1
    z = randn(23, n, v).to(TYPES[dtype]).cuda()
    z[:, -1] = 20.0
    u, tokens, p = rand(24, n).cuda(), torch.empty(n, dtype=torch.int64).cuda(), torch.empty(n).cuda()
    for _ in range(20):
        tokens.fill_(-7)
        cabi.sample(z, u, tokens, temperature=torch.zeros(n).cuda(), probabilities=p)
        assert (tokens == v - 1).all() and (p == 1).all()


def test_views_and_alignment():
    base, u = randn(12, 5, 3003), rand(13, 5)
    want = torch.empty(5, dtype=torch.int64)
    for z in (base[:, 1:], base[:, ::2], base[1:4, :2999], base.t().contiguous().t(), base.half()[:, 3:2001], base.flip(0)):
        n = z.shape[0]
        check(z if z.stride(1) >= 0 else z, u[:n], top_p=[0.8] * n, top_k=[100, 0, 30, 0, 5][:n])
    tokens = torch.full((10,), -7).cuda()  # every other place
    cabi.sample(base.cuda(), u.cuda(), tokens[::2], top_k=torch.full((10,), 5).cuda()[::2])
    cabi.sample(base.cuda(), u.cuda(), want := want.cuda(), top_k=torch.full((5,), 5).cuda())
    assert torch.equal(tokens[::2], want) and (tokens[1::2] == -7).all()
    cabi.sample(torch.empty(0, 10).cuda(), torch.empty(0).cuda(), torch.empty(0, dtype=torch.int64).cuda())


def test_the_largest_vocabulary_and_many_rows():
    z, u = randn(14, 2, 1 << 18) * 2.5, rand(15, 2)
    check(z, u, top_p=[0.9, 1.0], top_k=[0, 100000])
    n, v = 700, 999
    z, u = randn(16, n, v), rand(17, n)
    check(z, u, top_p=torch.full((n,), 0.9), top_k=torch.randint(0, 60, (n,), generator=torch.Generator().manual_seed(1)).to(torch.int32))


def test_the_same_bits_every_time_and_in_a_graph():
    z, u = (randn(18, 32, 50304) * 3).bfloat16().cuda(), rand(19, 32).cuda()
    p, k = torch.full((32,), 0.95).cuda(), torch.arange(32).cuda() * 200
    outs = []
    for _ in range(3):
        t, pr = torch.empty(32, dtype=torch.int64).cuda(), torch.empty(32).cuda()
        cabi.sample(z, u, t, top_p=p, top_k=k, probabilities=pr)
        outs.append((t, pr))
    assert all(torch.equal(a, b) for o in outs[1:] for a, b in zip(o, outs[0]))
    t, s = torch.zeros(32, dtype=torch.int64).cuda(), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        cabi.sample(z, u, t, top_p=p, top_k=k, stream=s.cuda_stream)
    u.copy_(rand(20, 32))
    graph.replay()
    want = torch.empty_like(t)
    torch.cuda.synchronize()
    cabi.sample(z, u, want, top_p=p, top_k=k)
    assert torch.equal(t, want)
