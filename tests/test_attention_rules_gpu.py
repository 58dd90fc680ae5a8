"""fml_attention_rules against a plain implementation in 64 bits; the bound is derived in serving_oracle.bound."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from fluidml_b200 import cabi
from serving_oracle import TYPES, attention, close


def randn(seed, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def visible_of(sq, sk, causal, prefix, qd, kd):
    at, key = torch.arange(sq)[:, None] + sk - sq, torch.arange(sk)[None, :]
    see = torch.ones(sq, sk, dtype=torch.bool)
    if causal:
        see = key <= at
        if prefix is not None:
            see = see | (key < prefix)
    if qd is not None:
        see = see & (qd[:, None] == kd[None, :])
    return see


def run(q, k, v, divisor=None, cap=0.0, causal=False, slopes=None, prefix=None, qd=None, kd=None, out=None, fill=7.0, heads=None):
    """Calls the operator on views as they are and holds every row of the given heads to the oracle."""
    b, h, sq, d = q.shape
    kv, sk = k.shape[1:3]
    divisor = divisor or math.sqrt(d)
    if out is None:
        out = torch.full((b, h, sq, d), fill, dtype=q.dtype).cuda()
    on = lambda x: None if x is None else x.cuda()  # noqa: E731
    cabi.attention_rules(q.cuda(), k.cuda(), v.cuda(), out, divisor, cap=cap, causal=causal, slopes=on(slopes), prefix=on(prefix),
                         q_documents=on(qd), k_documents=on(kd))
    cabi.check_device()
    got = out.cpu()
    for i in range(b):
        see = visible_of(sq, sk, causal, None if prefix is None else int(prefix[i]), None if qd is None else qd[i], None if kd is None else kd[i])
        for j in range(h) if heads is None else heads:
            bias = None
            if slopes is not None:
                bias = -slopes[j].double() * ((torch.arange(sq)[:, None] + sk - sq) - torch.arange(sk)[None, :]).abs().double()
            want, size = attention(q[i, j].cpu(), k[i, j * kv // h].cpu(), v[i, j * kv // h].cpu(), see, divisor, cap, bias)
            assert close(got[i, j], want, size, q.dtype), (i, j, float((got[i, j].double() - want).abs().max()))
    return got


SLOPES = torch.tensor([0.5, 0.25, 0.125, 0.0625])
LENGTHS = [(1, 1), (7, 7), (64, 64), (65, 63), (77, 77), (1, 200), (130, 40), (129, 257)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("d", [4, 32, 64, 80, 128])
@pytest.mark.parametrize("sq,sk", LENGTHS)
def test_lengths_and_head_sizes(dtype, d, sq, sk):
    t = TYPES[dtype]
    q, k, v = randn(1, 1, 2, sq, d, dtype=t), randn(2, 1, 1, sk, d, dtype=t), randn(3, 1, 1, sk, d, dtype=t)
    run(q, k, v)
    run(q, k, v, causal=True)  # more queries than keys: the first see nothing and are zero


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("cap", [0.0, 5.0, 50.0])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("kind", ["both", "causal", "prefix", "documents", "causal documents", "prefix documents"])
def test_rules_together(dtype, cap, bias, kind):
    t, b, s, d = TYPES[dtype], 2, 150, 64
    q, k, v = randn(4, b, 4, s, d, dtype=t) * 2, randn(5, b, 2, s, d, dtype=t), randn(6, b, 2, s, d, dtype=t)
    prefix = torch.tensor([0, 90], dtype=torch.int32) if "prefix" in kind else None
    docs = torch.stack((torch.repeat_interleave(torch.arange(4), torch.tensor([1, 70, 0, 79])[torch.tensor([0, 1, 3, 2])]),
                        torch.arange(s) % 3)) if "documents" in kind else None  # in a row, and interleaved
    run(q, k, v, cap=cap, causal=kind != "both" and kind != "documents", slopes=SLOPES if bias else None, prefix=prefix, qd=docs, kd=docs)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_queries_whose_document_has_no_key(dtype):
    t = TYPES[dtype]
    q, k, v = randn(7, 1, 2, 70, 64, dtype=t), randn(8, 1, 2, 140, 64, dtype=t), randn(9, 1, 2, 140, 64, dtype=t)
    qd = torch.arange(70)[None] // 10
    kd = torch.arange(140)[None] // 20 * 2  # the odd ones are missing
    got = run(q, k, v, qd=qd, kd=kd)
    assert (got[:, :, (qd[0] % 2 == 1)] == 0).all()
    run(q, k, v, qd=qd.to(torch.int32), kd=kd + (1 << 33))  # nothing seen at all, and numbers of either width
    run(q, k, torch.full_like(v, math.nan), qd=qd, kd=kd + (1 << 33))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_what_is_not_seen_adds_nothing(dtype, value):
    t, s = TYPES[dtype], 200
    q, k, v = randn(10, 1, 2, s, 64, dtype=t), randn(11, 1, 1, s, 64, dtype=t), randn(12, 1, 1, s, 64, dtype=t)
    docs = torch.zeros(1, s, dtype=torch.int32)
    docs[0, 150:] = 1
    for x in (k, v):
        kept = x.clone()
        x[0, 0, 150:160] = value  # seen by the second document alone
        out = torch.empty(1, 2, s, 64, dtype=t).cuda()
        cabi.attention_rules(q.cuda(), k.cuda(), v.cuda(), out, 8.0, causal=True, q_documents=docs.cuda(), k_documents=docs.cuda())
        for h in range(2):
            want, size = attention(q[0, h, :150], k[0, 0, :150], v[0, 0, :150], visible_of(150, 150, True, None, None, None), 8.0)
            assert close(out[0, h, :150], want, size, t)
        x.copy_(kept)
    v[0, 0, 20] = value  # seen by the later ones: theirs are not finite, the others' are as before
    cabi.attention_rules(q.cuda(), k.cuda(), v.cuda(), out, 8.0, causal=True)
    want, size = attention(q[0, 0, :20], k[0, 0, :20], v[0, 0, :20], visible_of(20, 20, True, None, None, None), 8.0)
    assert close(out[0, 0, :20], want, size, t) and not out[0, 0, 20:].isfinite().any()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("large", [2.0 ** 15, 2.0 ** 40, 2.0 ** 100])
def test_large_numbers_that_are_not_seen_cost_no_bits(dtype, d, large):
    """Keys and values of another document, and of later rows, in the tile of those that a row sees."""
    t, s = TYPES[dtype], 200
    large = min(large, 2.0 ** 15) if t == torch.float16 else large
    for which in range(2):
        q, k, v = randn(40, 1, 2, s, d, dtype=t), randn(41, 1, 1, s, d, dtype=t), randn(42, 1, 1, s, d, dtype=t)
        docs = torch.zeros(1, s, dtype=torch.int32)
        docs[0, 90:] = 1
        (k, v)[which][0, 0, 70:90] *= large
        run(q[:, :, 90:], k, v, qd=docs[:, 90:], kd=docs)                                # behind them
        out = torch.empty(1, 2, s, d, dtype=t).cuda()
        cabi.attention_rules(q.cuda(), k.cuda(), v.cuda(), out, math.sqrt(d), causal=True)
        want, size = attention(q[0, 0, :70], k[0, 0, :70], v[0, 0, :70], visible_of(70, 70, True, None, None, None), math.sqrt(d))
        assert close(out[0, 0, :70], want, size, t)                                      # in front of them


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("d", [64, 80, 128])
def test_what_is_not_finite_stays_in_its_feature(dtype, d):
    t, s, h = TYPES[dtype], 700, 12
    q, k, v = randn(43, 1, h, s, d, dtype=t), randn(44, 1, h // 3, s, d, dtype=t), randn(45, 1, h // 3, s, d, dtype=t)
    v[:, :, 33, 5] = math.inf
    out = torch.empty(1, h, s, d, dtype=t).cuda()
    slopes = torch.tensor([2.0 ** -(8 + i / 4) for i in range(h)])
    cabi.attention_rules(q.cuda(), k.cuda(), v.cuda(), out, math.sqrt(d), causal=True, slopes=slopes.cuda(), cap=30.0)
    other = torch.arange(d) != 5
    for j in (0, 7):
        bias = -slopes[j].double() * (torch.arange(s)[:, None] - torch.arange(s)[None, :]).abs().double()
        want, size = attention(q[0, j], k[0, j // 3][:], v[0, j // 3][:, other], visible_of(s, s, True, None, None, None), math.sqrt(d), 30.0, bias)
        assert close(out[0, j][:, other], want, size, t)
        assert (out[0, j, 33:, 5] == math.inf).all() and out[0, j, :33, 5].isfinite().all()
    for x in (q, k, v):
        y = [math.nan * z if z is x else z for z in (q, k, v)]
        cabi.attention_rules(*(z.cuda() for z in y), out, math.sqrt(d), causal=True)
        assert out.isnan().all()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_strides_and_alignment(dtype):
    t = TYPES[dtype]
    b, s, d = 2, 70, 64
    for make in (lambda x: x.transpose(1, 2).contiguous().transpose(1, 2),                      # heads are columns of the rows
                 lambda x: torch.cat((x, x[..., :1]), -1).contiguous()[..., :d],                # rows of 65
                 lambda x: torch.cat((x[..., :1], x), -1).contiguous()[..., 1:],                # and off the boundary
                 lambda x: x.transpose(2, 3).contiguous().transpose(2, 3)):                     # features outermost
        q, k, v = (make(randn(i, b, h, s, d, dtype=t)).cuda() for i, h in ((13, 4), (14, 2), (15, 2)))
        out = make(torch.zeros(b, 4, s, d, dtype=t)).cuda()
        if out.stride() != q.stride():
            out = torch.empty_strided(q.shape, q.stride(), dtype=t, device="cuda") if q.stride(3) != 1 or q.stride(2) == d else out
        run(q, k, v, causal=True, out=out)
    # one key and value for every batch and head, a documents row for every batch
    q, k, v = randn(16, b, 4, s, d, dtype=t), randn(17, 1, 1, s, d, dtype=t).expand(b, 2, s, d), randn(18, 1, 1, s, d, dtype=t).expand(b, 2, s, d)
    run(q, k, v, qd=(torch.arange(s) // 30).expand(b, s), kd=(torch.arange(s) // 30).expand(b, s))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 80, 128])
@pytest.mark.parametrize("kind", ["both", "causal", "prefix bias", "documents cap"])
def test_larger_problems(dtype, d, kind):
    """Sizes that the fifth-generation tensor cores take; two heads are held to the oracle."""
    t, b, s, h, kv = TYPES[dtype], 2, 1100, 16, 4
    q, k, v = randn(19, b, h, s, d, dtype=t), randn(20, b, kv, s, d, dtype=t), randn(21, b, kv, s, d, dtype=t)
    docs = torch.stack((torch.arange(s) // 300, (torch.arange(s) > 517).long())) if "documents" in kind else None
    slopes = torch.tensor([2.0 ** (-(i + 1) / 2) for i in range(h)]) if "bias" in kind else None
    run(q, k, v, cap=20.0 if "cap" in kind else 0.0, causal=kind != "both", slopes=slopes,
        prefix=torch.tensor([700, 0]) if "prefix" in kind else None, qd=docs, kd=docs, heads=(0, 13))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_larger_problems_with_rows_that_see_nothing_and_infinities(dtype):
    t, s, h, d = TYPES[dtype], 1300, 24, 64
    q, k, v = randn(22, 1, h, s, d, dtype=t), randn(23, 1, h, s, d, dtype=t), randn(24, 1, h, s, d, dtype=t)
    v[:, :, 1200:] = math.inf
    k[:, :, 1250:] = math.nan
    docs = torch.arange(s)[None] // 100
    qd = docs.clone()
    qd[:, 300:420] = 99  # see nothing
    qd[:, 1200:] = -1
    run(q, k, v, causal=True, qd=qd, kd=docs, heads=(0, 7))
    run(q, k[:, :, :900], v[:, :, :900], causal=True, heads=(3,))  # more queries than keys


@pytest.mark.parametrize("dtype,sk", [("f32", 131000), ("f32", 131200), ("f16", 262100), ("bf16", 262200)])
def test_long_rows_on_either_side_of_what_a_kernel_lists(dtype, sk):
    t = TYPES[dtype]
    q, k, v = randn(49, 1, 1, 128, 64, dtype=t), randn(50, 1, 1, sk, 64, dtype=t), randn(51, 1, 1, sk, 64, dtype=t)
    docs = (torch.arange(sk)[None] >= sk - 40000).to(torch.int32)
    run(q, k, v, causal=True, qd=torch.arange(128, dtype=torch.int32)[None] % 2, kd=docs)


@pytest.mark.parametrize("kind", ["plain", "bias", "documents"])
def test_sums_over_many_keys_in_fp32(kind):
    """Values of one sign, so that a context that is cut as it grows shows.  Small queries: scores sum |q||k| / 8 of 2 at most, so
    they are off by 12 x 2^-23 x 2 for the tensor core's instructions, 2^-20 x 2 for the split operands and 20 x 2^-23 for the bias:
    7.2e-6, twice in a weight.  The context: at most 16 blocks of 12 instructions lose 2^-23 each of what one accumulator holds,
    2.3e-5, and 20 sums in fp32 2^-24 each, 1.2e-6."""
    sq, sk, d = 130, 20000, 64
    q, k, v = randn(46, 1, 2, sq, d) * 0.1, randn(47, 1, 1, sk, d), randn(48, 1, 1, sk, d).abs() + 1
    slopes = torch.tensor([1e-3, 5e-4]) if kind == "bias" else None  # the largest score moves along the keys
    qd, kd = (torch.arange(sq)[None] % 3, torch.arange(sk)[None] // 300 % 2) if kind == "documents" else (None, None)  # 2: none
    out = torch.empty(1, 2, sq, 2 * d).cuda()[..., ::2] if kind == "documents" else torch.empty(1, 2, sq, d).cuda()
    on = lambda x: None if x is None else x.cuda()  # noqa: E731
    cabi.attention_rules(q.cuda(), k.cuda(), v.cuda(), out, 8.0, causal=True, slopes=on(slopes), q_documents=on(qd), k_documents=on(kd))
    cabi.check_device()
    see = visible_of(sq, sk, True, None, None if qd is None else qd[0], None if kd is None else kd[0])
    for h in range(2):
        distance = ((torch.arange(sq)[:, None] + sk - sq) - torch.arange(sk)[None, :]).abs().double()
        want, size = attention(q[0, h], k[0, 0], v[0, 0], see, 8.0, 0.0, None if slopes is None else -slopes[h].double() * distance)
        err = (out[0, h].cpu().double() - want).abs()
        assert (err <= (2 * 7.2e-6 + 2.3e-5 + 1.2e-6 + 1e-6) * size + 1e-7).all(), float((err / size.clamp_min(1e-30)).max())


@pytest.mark.parametrize("rows,stride", [(160, 64), (131, 64), (100, 66)])
def test_few_keys_go_to_one_accumulator(rows, stride):
    """fp32 of head size 64: scores of zero, so weights of one, and values of 21 bits, which pairs hold: nothing is rounded but sums.  The
    tensor cores cut 2^-25 of the sum so far on average, which is on average half of what it becomes, in each of the eight
    instructions of a block that add anything (the weights' low halves are zero): 4.8e-7 for the four blocks of an accumulator, however
    many follow.  2048 keys are 32 blocks.  Rows that end inside a warp's, and an output whose rows are not on 16 bytes."""
    n = 2048
    q, k = torch.zeros(1, 2, rows, 64), randn(70, 1, 1, n, 64)
    v = 1.0 + torch.randint(0, 1 << 20, (1, 1, n, 64), generator=torch.Generator().manual_seed(71)) / 2.0 ** 20
    out = torch.full((1, 2, rows, stride), 7.0).cuda()
    cabi.attention_rules(q.cuda(), k.cuda(), v.cuda(), out[..., :64], 8.0)
    cabi.check_device()
    want = v.double().mean(2, keepdim=True)
    error = (out[..., :64].double().cpu() - want) / want
    assert error.abs().max() <= 32 * 2.0 ** -23 + 10 * 2.0 ** -24  # if every instruction cut a whole unit; the roundings of eight folds
    assert abs(float(error.mean())) <= 32 * 2.0 ** -26 + 2.0 ** -24, float(error.mean())
    assert (out[..., 64:] == 7).all()


@pytest.mark.parametrize("kind", ["rising", "falling", "late documents"])
def test_contexts_that_wait_while_scales_and_maxima_move(kind):
    """fp32 of head size 64 over 21 blocks of keys: values whose scale changes by up to 2^40 from block to block, maxima that rise or fall
    by a few units a block, and rows whose first key comes after several accumulators."""
    n, h = 1340, 2
    q, k, v = randn(73, 1, h, n, 64), randn(74, 1, h, n, 64), randn(75, 1, h, n, 64)
    block = torch.arange(n) // 64
    exponents = torch.randint(-20, 21, (22,), generator=torch.Generator().manual_seed(76))
    v = v * (2.0 ** exponents[block].float())[:, None]
    q[..., 0], k[..., 0] = 8.0, (block if kind == "rising" else -block).float() * 3.0  # scores move by three a block
    documents = None
    if kind == "late documents":
        k[..., 0] = 0.0
        documents = torch.zeros(1, n, dtype=torch.int32)
        documents[:, 1000:] = torch.arange(n - 1000) % 3 + 1  # queries from 1000 on see nothing before
        documents[:, 40:44] = torch.tensor([1, 2, 3, 9])  # but for one key each
        documents[:, 1100] = 7  # and one sees itself alone
    run(q, k, v, causal=True, qd=documents, kd=documents)
    run(q[:, :, :70], k, v, qd=None if documents is None else documents[:, :70], kd=documents)


@pytest.mark.parametrize("dtype,d", [("f32", 80), ("f16", 64), ("f16", 96), ("f16", 128), ("bf16", 64), ("bf16", 128)])
@pytest.mark.parametrize("rows", [70, 1340])
def test_small_weights_beside_far_larger_values(dtype, d, rows):
    """Weights fall by e^-2 and more from block to block, values change by up to 2^24 (2^40 where the type holds that): what a small weight
    has lost would show.  Products of a score's sum reach 84, four times what the bound is derived for."""
    t, n, h = TYPES[dtype], 1340, 2
    q, k, v = randn(77, 1, h, rows, d), randn(78, 1, h, n, d), randn(79, 1, h, n, d)
    block = torch.arange(n) // 64
    reach = 12 if dtype == "f16" else 20
    exponents = torch.randint(-reach, reach + 1, (22,), generator=torch.Generator().manual_seed(80))
    q[..., 0], k[..., 0] = 8.0, -block.float() * 3.0
    q, k, v = q.to(t), k.to(t), (v * (2.0 ** exponents[block].float())[:, None]).to(t)
    out = torch.empty(1, h, rows, d, dtype=t).cuda()
    cabi.attention_rules(q.cuda(), k.cuda(), v.cuda(), out, math.sqrt(d), causal=True)
    cabi.check_device()
    step = torch.finfo(t).eps / 2
    see = visible_of(rows, n, True, None, None, None)
    for j in range(h):
        want, size = attention(q[0, j], k[0, j], v[0, j], see, math.sqrt(d))
        err = (out[0, j].double().cpu() - want).abs()
        weight = 4 * 3e-4 if t == torch.float32 else step + 4e-4
        assert (err <= weight * size + step * want.abs() + 1e-7).all(), float((err / size).max())


@pytest.mark.parametrize("length,d", [(700, 128), (300, 96), (10, 128)])
def test_how_far_fp32_is_off(length, d):
    """fp32 scores lose little of what the tensor cores cut.  N(0, 1) throughout, so q . k is some 11.3 and a partial sum of 32 features
    5.7: its four instructions cut 2^-25 of half of that each, 6e-8 of a score of one with four partial sums of either sign; five
    rounded steps 1.5e-7, the splits to 2^-22 of either operand 1.7e-7; in the context twelve instructions of 2^-25 of half the sum,
    1.8e-7, and the result's rounding 4e-8.  Together 3e-7 in the 2-norm; 5e-7 leaves room for few rows."""
    q, k, v = randn(81, 1, 4, length, d), randn(82, 1, 4, length, d), randn(83, 1, 4, length, d)
    out = torch.empty(1, 4, length, d).cuda()
    cabi.attention_rules(q.cuda(), k.cuda(), v.cuda(), out, math.sqrt(d), causal=True)
    cabi.check_device()
    want = torch.stack([attention(q[0, h], k[0, h], v[0, h], visible_of(length, length, True, None, None, None), math.sqrt(d))[0] for h in range(4)])
    assert float((out[0].double().cpu() - want).norm() / want.norm()) <= 5e-7


def test_large_scores():
    """Scores of hundreds: the running maximum moves, and weights of distant keys vanish."""
    for dtype in TYPES.values():
        q, k, v = randn(25, 1, 2, 300, 64, dtype=dtype) * 16, randn(26, 1, 2, 300, 64, dtype=dtype), randn(27, 1, 2, 300, 64, dtype=dtype)
        out = torch.empty(1, 2, 300, 64, dtype=dtype).cuda()
        cabi.attention_rules(q.cuda(), k.cuda(), v.cuda(), out, 8.0, causal=True)
        for h in range(2):
            want, size = attention(q[0, h], k[0, h], v[0, h], visible_of(300, 300, True, None, None, None), 8.0)
            # scores sixteen times as large as the bound is derived for
            step = torch.finfo(dtype).eps / 2
            assert ((out[0, h].double().cpu() - want).abs() <= (step * (dtype != torch.float32) + 16 * 3e-4) * size + step * want.abs() + 1e-7).all()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("d", [64, 80, 128])
@pytest.mark.parametrize("cap,divisor", [(2.0 ** 64, 8.0), (2.0 ** -64, 8.0), (50.0, 2.0 ** 120), (30.0, -8.0)])
def test_factors_at_their_ends(dtype, d, cap, divisor):
    """A cap that changes nothing, one that makes all scores alike, a divisor that does."""
    q, k, v = (randn(60 + i, 1, 2, 300, d, dtype=TYPES[dtype]) for i in range(3))
    run(q, k, v, divisor=divisor, cap=cap, causal=True)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("bias", [False, True])
def test_scores_beyond_the_cap(dtype, d, bias):
    """Scores of up to some 70, a cap of 10: most lie where tanh is flat, some in its bend, over more keys than a tile has."""
    t, n, cap = TYPES[dtype], 2100, 10.0
    q, k, v = randn(63, 1, 4, n, d, dtype=t) * 16, randn(64, 1, 2, n, d, dtype=t), randn(65, 1, 2, n, d, dtype=t)
    out = torch.empty(1, 4, n, d, dtype=t).cuda()
    cabi.attention_rules(q.cuda(), k.cuda(), v.cuda(), out, math.sqrt(d), cap=cap, causal=True, slopes=SLOPES.cuda() if bias else None)
    cabi.check_device()
    rows = torch.cat((torch.arange(0, n, 97), torch.tensor([n - 1])))
    step = torch.finfo(t).eps / 2
    for h in (0, 3):
        distance = (rows[:, None] - torch.arange(n)).abs().double()
        want, size = attention(q[0, h, rows], k[0, h // 2], v[0, h // 2], torch.arange(n) <= rows[:, None], math.sqrt(d), cap,
                               -SLOPES[h].double() * distance if bias else None)
        err = (out[0, h, rows].double().cpu() - want).abs()
        # scores sixteen times as large as the bound is derived for, which the cap only brings nearer to one another; beside it the cap's
        # own 2.4e-7 of 10, and a bias of up to 1050 in steps of 2^-24 of it, each twice (numerator and sum)
        weight = step * (t != torch.float32) + 16 * 3e-4 + 2 * 2.4e-6 + (2 * 9 * 1050 * 1.4427 * 2.0 ** -24 if bias else 0.0)
        assert (err <= weight * size + step * want.abs() + 1e-7).all(), float(err.max())


def test_two_streams_and_a_captured_graph():
    t = torch.bfloat16
    x = [(randn(30 + i, 1, 8, 1000, 64, dtype=t).cuda(), randn(40 + i, 1, 8, 1000, 64, dtype=t).cuda()) for i in range(2)]
    want = [torch.empty_like(q) for q, _ in x]
    for (q, k), o in zip(x, want):
        cabi.attention_rules(q, k, k, o, 8.0, causal=True)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in x], [torch.empty_like(q) for q, _ in x]
    for _ in range(10):
        for (q, k), o, s in zip(x, outs, streams):
            cabi.attention_rules(q, k, k, o, 8.0, causal=True, stream=s.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, outs))
    graph, out = torch.cuda.CUDAGraph(), torch.zeros_like(want[0])
    q, k = (a.clone() for a in x[0])
    s = streams[0]
    with torch.cuda.graph(graph, stream=s):
        cabi.attention_rules(q, k, k, out, 8.0, causal=True, stream=s.cuda_stream)
    q.copy_(x[1][0]); k.copy_(x[1][1])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want[1])


def test_empty():
    e = torch.empty(0, 2, 5, 64).cuda()
    cabi.attention_rules(e, e, e, e.clone(), 8.0)
    q, k = torch.ones(1, 2, 5, 64).cuda(), torch.empty(1, 2, 0, 64).cuda()
    out = torch.full_like(q, 7)
    cabi.attention_rules(q, k, k, out, 8.0)
    assert (out == 0).all()  # no key: zeros
    cabi.attention_rules(torch.empty(1, 2, 0, 64).cuda(), q, q, torch.empty(1, 2, 0, 64).cuda(), 8.0)
