"""The serving operators as they are used: a prompt (positions and append, attention by rules, a token), then rounds of drafted
tokens (positions and append, attention of the tree over the cache, a token for each draft), held to 64 bits end to end; and what
no test of a single operator calls.

Tolerance of the chain: queries, keys and values are rounded once on the way in (half a step each of a turned value, 2^-11 for fp16);
a score of 7 sums |q||k| / divisor (serving_oracle.bound) is then off by 2 x 2^-11 x 7 at most more, twice that in a weight.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from fluidml_b200 import cabi
from fluidml_b200.cabi import DeviceTensor as DT
from serving_oracle import HALF_STEP, TYPES, attention, bound, sample as sample_oracle

I32 = torch.int32


def turned(x, positions, f):
    """Halves convention over all features, 64 bits."""
    x = x.double()
    angle = positions.double()[:, None, None] * f.double()
    a, b = x.chunk(2, -1)
    return torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()), -1)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_a_prompt_and_two_rounds_of_drafts(dtype):
    t, heads, kv, d, page, vocab = TYPES[dtype], 4, 2, 64, 16, 1000
    g = torch.Generator().manual_seed(1)
    randn = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    f = torch.from_numpy(cabi.rotary_frequencies(d, cabi.ROTARY_LINEAR, factor=2.0)[0])
    unembed = randn(heads * d, vocab) * 0.2
    lengths = [37, 150]  # two prompts, the second attended to with a prefix of 40
    table = torch.randperm(40, generator=g).reshape(2, 20).to(I32)
    k_cache, v_cache = (torch.zeros(40, page, kv, d, dtype=t).cuda() for _ in range(2))
    cached = [[], []]  # what the oracle keeps: (turned key, value) in 64 bits
    slot = lambda r, i: int(table[r, i // page]) * page + i % page  # noqa: E731
    space = torch.empty(32 << 20, dtype=torch.uint8).cuda()
    extra = 4 * HALF_STEP[t] * 7

    def step(q, k, v, positions, slots):
        q_out = torch.empty_like(q).cuda()
        cabi.rotary_positions(q.cuda(), k.cuda(), v.cuda(), positions.cuda(), torch.tensor(slots).cuda(), f.cuda(), q_out, k_cache, v_cache)
        return q_out

    def hold(got, want, size):
        err = (got.double().cpu() - want).abs()
        assert (err <= bound(t, size, want) + extra * size).all(), float(err.max())

    def choose(context, want):
        """Tokens from the context's logits; the same random number through the oracle on the kernel's own logits."""
        logits = (context.float().flatten(1) @ unembed.cuda()).to(t)
        u, n = torch.rand(len(want), generator=g), len(want)
        tokens, top_p, top_k = torch.empty(n, dtype=torch.int64).cuda(), torch.full((n,), 0.9).cuda(), torch.full((n,), 50, dtype=I32).cuda()
        cabi.sample(logits, u.cuda(), tokens, top_p=top_p, top_k=top_k)
        for i in range(n):
            token, _, near = sample_oracle(logits[i].float().tolist(), u[i].item(), 1.0, 50, torch.tensor(0.9).item(), 0.0)
            assert near < 1e-9 or tokens[i].item() == token

    for r, n in enumerate(lengths):
        q, k, v = (randn(n, h, d).to(t) for h in (heads, kv, kv))
        positions = torch.arange(n)
        q_out = step(q, k, v, positions, [slot(r, i) for i in range(n)])
        places = torch.tensor([slot(r, i) for i in range(n)]).cuda()
        kk, vv = (x.flatten(0, 1)[places][None].transpose(1, 2) for x in (k_cache, v_cache))  # the prompt's keys as they lie in the cache
        prefix = torch.tensor([40 * r], dtype=I32).cuda()
        out = torch.empty(1, n, heads, d, dtype=t).cuda().transpose(1, 2)
        cabi.attention_rules(q_out[None].transpose(1, 2), kk, vv, out, math.sqrt(d), causal=True, prefix=prefix)
        qt, kt = turned(q, positions, f), turned(k, positions, f)
        cached[r] = [kt, v.double()]
        key, at = torch.arange(n)[None, :], torch.arange(n)[:, None]
        for h in range(heads):
            want, size = attention(qt[:, h], kt[:, h // 2], v[:, h // 2], (key <= at) | (key < 40 * r), math.sqrt(d))
            hold(out[0, h], want, size)
        choose(out[0].transpose(0, 1)[-1:], [0])
    for drafts in ([3, 5], [1, 2]):
        contexts = [len(c[0]) for c in cached]
        masks, depths = [], []
        for n in drafts:  # a first token, the others its children or grandchildren
            m = []
            for j in range(n):
                m.append((m[(j - 1) // 2] if j else 0) | 1 << j)
            masks += m
            depths.append([bin(x).count("1") - 1 for x in m])
        tokens = sum(drafts)
        q, k, v = (randn(tokens, h, d).to(t) for h in (heads, kv, kv))
        positions = torch.tensor([c + e for c, ds in zip(contexts, depths) for e in ds])
        slots = [slot(r, contexts[r] + j) for r in range(2) for j in range(drafts[r])]
        q_out = step(q, k, v, positions, slots)
        out = torch.empty(tokens, heads, d, dtype=t).cuda()
        start = torch.tensor([0, drafts[0], tokens], dtype=I32).cuda()
        cabi.attention_tree(q_out, k_cache, v_cache, table.cuda(), torch.tensor(contexts, dtype=I32).cuda(), start, torch.tensor(masks).cuda(), out,
                            space, math.sqrt(d))
        cabi.check_device()
        qt, kt = turned(q, positions, f), turned(k, positions, f)
        for r in range(2):
            a, n = sum(drafts[:r]), drafts[r]
            keys, values = torch.cat((cached[r][0], kt[a:a + n])), torch.cat((cached[r][1], v[a:a + n].double()))
            see = torch.cat((torch.ones(n, contexts[r], dtype=torch.bool),
                             torch.tensor([[masks[a + i] >> j & 1 for j in range(n)] for i in range(n)], dtype=torch.bool)), 1)
            for h in range(heads):
                want, size = attention(qt[a:a + n, h], keys[:, h // 2], values[:, h // 2], see, math.sqrt(d))
                hold(out[a:a + n, h], want, size)
            cached[r] = [keys[:contexts[r] + 1], values[:contexts[r] + 1]]  # the first draft is accepted
        choose(out, range(tokens))


def test_arrays_of_the_bindings_own():
    """The same calls on DeviceTensors, as a program without torch makes them."""
    g = torch.Generator().manual_seed(2)
    x = torch.randn(6, 2, 64, generator=g)
    f = cabi.rotary_frequencies(64)[0]
    out = DT((6, 2, 64), "float32")
    cabi.rotary_positions(DT.from_numpy(x.numpy()), None, None, DT.from_numpy(torch.arange(6).numpy()), None, DT.from_numpy(f), out, None, None)
    want = turned(x, torch.arange(6), torch.from_numpy(f))
    assert (torch.from_numpy(out.numpy()).double() - want).abs().max() <= 2e-6 * x.abs().max()
    q = torch.randn(1, 2, 6, 64, generator=g)
    o = DT((1, 2, 6, 64), "float32")
    cabi.attention_rules(*(DT.from_numpy(q.numpy()) for _ in range(3)), o, 8.0, causal=True)
    for h in range(2):
        want, size = attention(q[0, h], q[0, h], q[0, h], torch.ones(6, 6).tril().bool(), 8.0)
        assert ((torch.from_numpy(o.numpy())[0, h].double() - want).abs() <= bound(torch.float32, size, want)).all()
    z = torch.randn(3, 500, generator=g)
    tokens = DT((3,), "int64")
    cabi.sample(DT.from_numpy(z.numpy()), DT.from_numpy(torch.zeros(3).numpy()), tokens, temperature=DT.from_numpy(torch.zeros(3).numpy()))
    assert tokens.numpy().tolist() == z.argmax(-1).tolist()
    cache = torch.randn(3, 16, 2, 64, generator=g)
    space = cabi.DeviceBuffer(cabi.attention_tree_workspace(1, 1, 2, 2, 64))
    one = lambda *v: DT.from_numpy(torch.tensor(v, dtype=I32).numpy())  # noqa: E731
    o = DT((1, 2, 64), "float32")
    c = DT.from_numpy(cache.numpy())
    cabi.attention_tree(DT.from_numpy(x[:1].numpy()), c, c, DT.from_numpy(torch.tensor([[2, 0, 1]], dtype=I32).numpy()), one(40), one(0, 1), None, o, space, 8.0)
    keys = cache[[2, 0, 1]].flatten(0, 1)[:41]
    for h in range(2):
        want, size = attention(x[:1, h], keys[:, h], keys[:, h], torch.ones(1, 41).bool(), 8.0)
        assert ((torch.from_numpy(o.numpy())[:, h].double() - want).abs() <= bound(torch.float32, size, want)).all()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("cap", [0.0, 10.0])
@pytest.mark.parametrize("length", [90, 600])
def test_a_negative_divisor(dtype, cap, length):
    t = TYPES[dtype]
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(1, 2, length, 64, generator=g).to(t) for _ in range(3))
    out = torch.empty_like(q).cuda()
    cabi.attention_rules(q.cuda(), k.cuda(), v.cuda(), out, -8.0, cap=cap, causal=True)
    for h in range(2):
        want, size = attention(q[0, h], k[0, h], v[0, h], torch.ones(length, length).tril().bool(), -8.0, cap)
        assert ((out[0, h].double().cpu() - want).abs() <= bound(t, size, want)).all()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("kind", ["narrow", "wide", "far", "mixed", "farthest"])
@pytest.mark.parametrize("causal", [False, True])
def test_documents_of_any_width_over_long_rows(dtype, kind, causal):
    t, s = TYPES[dtype], 700
    g = torch.Generator().manual_seed(4)
    q, k, v = (torch.randn(1, 2, s, 64, generator=g).to(t) for _ in range(3))
    docs = torch.bucketize(torch.arange(s), torch.tensor([1, 129, 256, 300, 513, 640]), right=True)
    if kind == "far":  # differences beyond 32 bits, in both directions, and two that differ in the upper half alone
        docs = torch.tensor([0, 1 << 40, -(1 << 40), (1 << 40) + 5, 1 << 33, 1 << 34, 7])[docs]
    elif kind == "farthest":
        docs = torch.tensor([-(1 << 63), (1 << 63) - 1, 0, -1, 1, (1 << 63) - 2, -(1 << 63) + 1])[docs]
    qd, kd = docs[None], docs[None]
    if kind == "narrow":
        qd, kd = qd.to(I32), kd.to(I32)
    elif kind == "mixed":
        kd = kd.to(I32)
    out = torch.empty_like(q).cuda()
    cabi.attention_rules(q.cuda(), k.cuda(), v.cuda(), out, 8.0, causal=causal, q_documents=qd.cuda(), k_documents=kd.cuda())
    cabi.check_device()
    see = docs[:, None] == docs[None, :]
    if causal:
        see &= torch.ones(s, s).tril().bool()
    for h in range(2):
        want, size = attention(q[0, h], k[0, h], v[0, h], see, 8.0)
        assert ((out[0, h].double().cpu() - want).abs() <= bound(t, size, want)).all()


def test_scattered_documents_and_disjoint_tiles():
    """Query tiles of one CTA whose keys lie far apart: their products wait for different tiles of keys."""
    for d in (64, 128):
        t, sq, sk = torch.bfloat16, 512, 6000
        g = torch.Generator().manual_seed(5)
        q, k, v = torch.randn(1, 2, sq, d, generator=g).to(t), torch.randn(1, 2, sk, d, generator=g).to(t), torch.randn(1, 2, sk, d, generator=g).to(t)
        kd = torch.arange(sk) // 1000
        for order in ([0, 5, 2, 2], [5, 0, 1, 4], [3, 9, 9, 0]):  # by tile of 128 queries; 9: none
            qd = torch.tensor(order).repeat_interleave(128)
            out = torch.empty_like(q).cuda()
            cabi.attention_rules(q.cuda(), k.cuda(), v.cuda(), out, math.sqrt(d), q_documents=qd[None].cuda(), k_documents=kd[None].cuda())
            cabi.check_device()
            want, size = attention(q[0, 1], k[0, 1], v[0, 1], qd[:, None] == kd[None, :], math.sqrt(d))
            assert ((out[0, 1].double().cpu() - want).abs() <= bound(t, size, want)).all()


def test_tensors_the_calls_refuse():
    x = torch.zeros(2, 2, 64).cuda()
    with pytest.raises(cabi.FmlError):  # host memory
        cabi.rotary_positions(torch.zeros(2, 2, 64), None, None, torch.arange(2).cuda(), None, torch.ones(8).cuda(), x, None, None)
    with pytest.raises(cabi.FmlError):  # a type no kernel takes
        cabi.rotary_positions(x.double(), None, None, torch.arange(2).cuda(), None, torch.ones(8).cuda(), x.double(), None, None)
    with pytest.raises(cabi.FmlError):  # a position per token is missing
        cabi.rotary_positions(x, None, None, torch.arange(3).cuda(), None, torch.ones(8).cuda(), x.clone(), None, None)
    with pytest.raises(cabi.FmlError):  # in place through another view
        cabi.rotary_positions(x, None, None, torch.arange(2).cuda(), None, torch.ones(8).cuda(), x.transpose(0, 1), None, None)
    with pytest.raises(TypeError):
        cabi.rotary_positions(x, None, None, torch.arange(2).cuda(), None, torch.ones(8).cuda(), x.clone(), None, None, magnitude="1")
    cabi.check_device()


def spread(x, step=(1 << 31) + 64):
    """A copy of x whose first dim moves by more than 2^31 elements."""
    view = torch.empty((x.shape[0] - 1) * step + x[0].numel(), dtype=x.dtype, device="cuda").as_strided(x.shape, (step,) + x[0].contiguous().stride())
    return view.copy_(x)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_offsets_that_pass_32_bits(dtype):
    """The same bits as from tensors that lie together, which the other tests hold to 64 bits."""
    t = TYPES[dtype]
    rand = lambda seed, *s: torch.randn(s, generator=torch.Generator().manual_seed(seed)).to(t).cuda()  # noqa: E731
    # positions and append: far tokens, far pages
    q, k, v = rand(1, 2, 4, 64), rand(2, 2, 2, 64), rand(3, 2, 2, 64)
    at, slots, f = torch.tensor([5, 9]).cuda(), torch.tensor([7, 1]).cuda(), torch.logspace(0, -3, 32).cuda()
    kc, vc = rand(4, 2, 4, 2, 64), rand(5, 2, 4, 2, 64)
    far_k, far_v, far_out, out = spread(kc), spread(vc), spread(q), torch.empty_like(q)
    cabi.rotary_positions(q, k, v, at, slots, f, out, kc, vc)
    cabi.rotary_positions(spread(q), k, v, at, slots, f, far_out, far_k, far_v)
    assert torch.equal(out, far_out) and torch.equal(kc, far_k) and torch.equal(vc, far_v)
    # the cache read again; values as far as keys, and not
    table, context, start = (torch.tensor(x, dtype=I32).cuda() for x in ([[1, 0]], [6], [0, 2]))
    ws = torch.empty(cabi.attention_tree_workspace(1, 2, 4, 2, 64), dtype=torch.uint8).cuda()
    cabi.attention_tree(q, kc, vc, table, context, start, None, out, ws, 8.0)
    for cache in (far_v, vc):
        far_out.zero_()
        cabi.attention_tree(q, far_k, cache, table, context, start, None, far_out, ws, 8.0)
        assert torch.equal(out, far_out)
    del far_k, far_v, far_out
    # prompts of either size of kernel, batches far apart
    for s, d in ((40, 64), (1100, 64), (1100, 128)):
        q, k, v = rand(6, 2, 8, s, d), rand(7, 2, 4, s, d), rand(8, 2, 4, s, d)
        out, far_out = torch.empty_like(q), spread(torch.zeros_like(q))
        cabi.attention_rules(q, k, v, out, math.sqrt(d), causal=True)
        cabi.attention_rules(spread(q), k, v, far_out, math.sqrt(d), causal=True)
        assert torch.equal(out, far_out)
        far_out.zero_()
        cabi.attention_rules(q, spread(k), spread(v), far_out, math.sqrt(d), causal=True)
        assert torch.equal(out, far_out)
    # logits
    z, u = rand(9, 2, 5000), torch.tensor([0.3, 0.8]).cuda()
    token, far_token, p = torch.empty(2, dtype=I32).cuda(), torch.empty(2, dtype=I32).cuda(), torch.tensor([0.9, 0.9]).cuda()
    cabi.sample(z, u, token, top_p=p)
    cabi.sample(spread(z), u, far_token, top_p=p)
    assert torch.equal(token, far_token)
    cabi.check_device()
