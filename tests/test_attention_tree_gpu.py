"""fml_attention_tree against a plain implementation in 64 bits; the bound is derived in serving_oracle.bound."""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

from fluidml_b200 import cabi
from serving_oracle import TYPES, attention, close


def randn(seed, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


class Case:
    """Requests with ragged contexts over a shuffled paged cache; `drafts` new tokens each."""

    def __init__(self, contexts, drafts, heads, kv, d, page, dtype, tree, seed=0, spare=3):
        rng = random.Random(seed)
        self.contexts, self.drafts, self.page, self.kv, self.heads, self.d = contexts, drafts, page, kv, heads, d
        need = [-(-(c + n) // page) for c, n in zip(contexts, drafts)]
        order = list(range(sum(need) + 2))
        rng.shuffle(order)
        self.table = torch.full((len(contexts), max(max(need), 1) + 1), 0, dtype=torch.int32)
        at = 0
        for r, n in enumerate(need):
            self.table[r, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
            at += n
        self.k, self.v = (randn(seed + i, len(order), page, kv, d, dtype=dtype) for i in (1, 2))
        self.tokens = sum(drafts) + spare  # rows behind the last request
        self.q = randn(seed + 3, self.tokens, heads, d, dtype=dtype)
        self.start = torch.tensor([sum(drafts[:r]) for r in range(len(drafts) + 1)], dtype=torch.int32)
        self.tree = None
        if tree:
            self.tree = torch.zeros(self.tokens, dtype=torch.int64)
            for r, n in enumerate(drafts):
                masks = []
                for j in range(n):
                    parent = rng.randint(-1, j - 1)
                    masks.append((masks[parent] if parent >= 0 else 0) | (1 << j if j < 63 else -(1 << 63)))
                    self.tree[int(self.start[r]) + j] = masks[-1]

    def call(self, cap=0.0, slopes=None, stream=None, out=None, workspace=None):
        on = lambda x: None if x is None else x.cuda()  # noqa: E731
        if out is None:
            out = torch.full((self.tokens, self.heads, self.d), 7.0, dtype=self.q.dtype).cuda()
        if workspace is None:
            workspace = torch.empty(cabi.attention_tree_workspace(len(self.contexts), self.tokens, self.heads, self.kv, self.d), dtype=torch.uint8).cuda()
        cabi.attention_tree(on(self.q), on(self.k), on(self.v), on(self.table), torch.tensor(self.contexts, dtype=torch.int32).cuda(), on(self.start),
                            on(self.tree), out, workspace, math.sqrt(self.d), cap=cap, slopes=on(slopes), stream=stream)
        return out

    def rows(self, r, head):
        """(queries, keys, values, visible, distances) of a request and head."""
        a, n, c = int(self.start[r]), self.drafts[r], self.contexts[r]
        k, v = (x[self.table[r].long()].flatten(0, 1)[:c + n, head * self.kv // self.heads] for x in (self.k, self.v))
        j = torch.arange(n)
        if self.tree is None:
            fresh = j[None, :] <= j[:, None]
        else:
            fresh = torch.tensor([[int(self.tree[a + i]) >> b & 1 if b < 64 else 0 for b in range(n)] for i in range(n)], dtype=torch.bool).reshape(n, n)
        depth = fresh.sum(1) - 1
        at = torch.cat((torch.arange(c), c + depth))
        return self.q[a:a + n, head], k, v, torch.cat((torch.ones(n, c, dtype=torch.bool), fresh), 1), ((c + depth)[:, None] - at[None, :]).abs()

    def check(self, out, cap=0.0, slopes=None, heads=None):
        got = out.cpu()
        for r in range(len(self.contexts)):
            for h in range(self.heads) if heads is None else heads:
                q, k, v, see, distance = self.rows(r, h)
                want, size = attention(q, k, v, see, math.sqrt(self.d), cap, None if slopes is None else -slopes[h].double() * distance.double())
                a = int(self.start[r])
                assert close(got[a:a + len(want), h], want, size, self.q.dtype), (r, h, float((got[a:a + len(want), h].double() - want).abs().max()))
        behind = got[int(self.start[-1]):]
        assert (behind == 7).all()  # left as they were


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("d,heads,kv,page", [(64, 4, 4, 16), (128, 8, 2, 64), (80, 6, 1, 24), (8, 2, 2, 1)])
@pytest.mark.parametrize("drafts", [[1, 1, 1, 1], [5, 1, 7, 3], [16, 33, 2, 64]])
def test_types_heads_pages_and_trees(dtype, d, heads, kv, page, drafts):
    contexts = [0, 1, 130, 700]
    slopes = torch.tensor([2.0 ** (-i - 1) for i in range(heads)])
    for tree in (False, True):
        c = Case(contexts, drafts, heads, kv, d, page, TYPES[dtype], tree, seed=len(drafts) + d)
        c.check(c.call())
        c.check(c.call(cap=10.0, slopes=slopes), 10.0, slopes)
        cabi.check_device()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_pages_that_end_inside_a_tile_and_every_length(dtype):
    contexts = [0, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 191, 192, 193]
    c = Case(contexts, [1 + i % 3 for i in range(16)], 4, 1, 64, 16, TYPES[dtype], False, seed=7)
    c.check(c.call())


def test_many_requests_and_requests_without_new_tokens():
    rng = random.Random(3)
    contexts = [rng.choice((0, 3, 40, 300)) for _ in range(300)]
    drafts = [rng.choice((0, 1, 1, 2, 4)) for _ in range(300)]
    c = Case(contexts, drafts, 2, 1, 64, 16, torch.bfloat16, True, seed=9)
    c.check(c.call())


def test_one_long_request_among_short_ones():
    for dtype in TYPES.values():
        c = Case([20000, 5, 0, 333], [4, 1, 2, 3], 4, 2, 128, 32, dtype, True, seed=11)
        c.check(c.call(), heads=(0, 3))


def test_chains_longer_than_64():
    c = Case([100, 0], [150, 70], 4, 2, 64, 16, torch.float16, False, seed=13)
    c.check(c.call())
    tree = Case([100, 0], [150, 70], 4, 2, 64, 16, torch.float16, True, seed=13)
    tree.tree[64:150] = -1  # bits for the first 64 alone: later tokens are seen by no one
    tree.tree[150 + 64:] = 5
    tree.check(tree.call())


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("contexts,drafts,heads,kv", [([1340], [1], 4, 1), ([1340, 200, 700], [5, 1, 9], 4, 2), ([1340, 1300], [40, 30], 4, 1)])
def test_small_weights_beside_far_larger_values(dtype, contexts, drafts, heads, kv):
    """Weights fall by e^-2 from page to page, values change by up to 2^24 (2^40 where the type holds that); parts of a request's keys are
    joined.  Products of a score's sum reach 84, four times what the bound is derived for."""
    t, d, page = TYPES[dtype], 128, 64
    c = Case(contexts, drafts, heads, kv, d, page, torch.float32, False, seed=50)
    reach = 12 if dtype == "f16" else 20
    exponents = torch.randint(-reach, reach + 1, (24,), generator=torch.Generator().manual_seed(51)).float()
    c.q[..., 0] = 8.0
    for r in range(len(contexts)):
        for b in range(-(-(contexts[r] + drafts[r]) // page)):
            c.k[c.table[r, b], ..., 0] = -3.0 * b
            c.v[c.table[r, b]] *= 2.0 ** exponents[b]
    c.q, c.k, c.v = c.q.to(t), c.k.to(t), c.v.to(t)
    got = c.call().double().cpu()
    cabi.check_device()
    step = torch.finfo(t).eps / 2
    for r in range(len(contexts)):
        for h in range(heads):
            q, k, v, see, _ = c.rows(r, h)
            want, size = attention(q, k, v, see, math.sqrt(d))
            a = int(c.start[r])
            err = (got[a:a + len(want), h] - want).abs()
            weight = 4 * 3e-4 if t == torch.float32 else step + 4e-4
            assert (err <= weight * size + step * want.abs() + 1e-7).all(), (r, h, float((err / size).max()))


@pytest.mark.parametrize("contexts,drafts,heads,kv", [([258, 100, 31, 200, 90, 150], [1] * 6, 2, 2), ([700, 300], [20, 9], 4, 1)])
def test_how_far_fp32_is_off(contexts, drafts, heads, kv):
    """fp32 scores lose little of what the tensor cores cut.  N(0, 1) throughout, so q . k is some 11.3 and a partial sum of 32 features
    5.7: its four instructions cut 2^-25 of half of that each, 6e-8 of a score of one with four partial sums of either sign; five
    rounded steps 1.5e-7, the splits to 2^-22 of either operand 1.7e-7; in the context twelve instructions of 2^-25 of half the sum,
    1.8e-7, and the result's rounding 4e-8.  Together 3e-7 in the 2-norm; 5e-7 leaves room for few rows."""
    c = Case(contexts, drafts, heads, kv, 128, 16, torch.float32, False, seed=52)
    got = c.call().double().cpu()
    cabi.check_device()
    err = size = 0.0
    for r in range(len(contexts)):
        for h in range(heads):
            q, k, v, see, _ = c.rows(r, h)
            want, a = attention(q, k, v, see, math.sqrt(128))[0], int(c.start[r])
            err += float((got[a:a + len(want), h] - want).square().sum())
            size += float(want.square().sum())
    assert math.sqrt(err / size) <= 5e-7, math.sqrt(err / size)


def test_tokens_that_see_nothing():
    for dtype in TYPES.values():
        c = Case([0, 0, 9], [3, 2, 2], 2, 2, 64, 16, dtype, True, seed=15)
        c.tree[:] = 0
        out = c.call()
        c.check(out)
        assert (out[:5] == 0).all()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_what_is_not_seen_adds_nothing(dtype, value):
    c = Case([100, 1000], [4, 6], 4, 2, 64, 16, TYPES[dtype], True, seed=17)
    # beyond the requests' ends, and other requests' pages
    used = torch.zeros(c.k.shape[0], c.page, dtype=torch.bool)
    for r in range(2):
        for i in range(c.contexts[r] + c.drafts[r]):
            used[c.table[r, i // c.page], i % c.page] = True
    for x in (c.k, c.v):
        x[~used] = value
    c.check(c.call())
    # a draft that the others do not see
    for i in range(6):
        c.tree[4 + i] = 1 << i
    place = 1002
    c.v[c.table[1, place // c.page], place % c.page] = value
    out = c.call().cpu()
    for i in (0, 1, 3, 4, 5):
        q, k, v, see, _ = c.rows(1, 1)
        want, size = attention(q[i:i + 1], k, v, see[i:i + 1], 8.0)
        assert close(out[4 + i:5 + i, 1], want, size, c.q.dtype)
    assert not out[6].isfinite().any()


def test_bad_pages_lengths_and_ranges_are_left_out_and_recorded():
    c = Case([40, 50], [2, 2], 2, 2, 64, 16, torch.float32, False, seed=19)
    c.table[0, 1] = 10 ** 6  # keys 16 .. 31 are not there
    out = c.call().cpu()
    with pytest.raises(cabi.FmlError) as e:
        cabi.check_device()
    assert e.value.status == 7
    c.table[0, 1] = 0
    for h in range(2):
        for r, gone in ((0, slice(16, 32)), (1, slice(0, 0))):
            q, k, v, see, _ = c.rows(r, h)
            see[:, gone] = False
            want, size = attention(q, k, v, see, 8.0)
            assert close(out[2 * r:2 * r + 2, h], want, size, c.q.dtype)
    for change in ("context", "start", "negative"):
        c = Case([40, 50], [2, 2], 2, 2, 64, 16, torch.float32, False, seed=19)
        if change == "context":
            c.contexts = [40, 10 ** 9]
        elif change == "negative":
            c.contexts = [40, -5]
        else:
            c.start[2] = 1000
        good = Case([40, 50], [2, 2], 2, 2, 64, 16, torch.float32, False, seed=19).call()
        assert torch.equal(c.call()[:2], good[:2])  # the other request is as it was
        with pytest.raises(cabi.FmlError):
            cabi.check_device()
        cabi.check_device()


def test_strides():
    c = Case([70, 300], [3, 2], 4, 2, 64, 16, torch.bfloat16, True, seed=21)
    want = c.call()
    c.k, c.v = torch.stack((c.k, c.v), 1).unbind(1)  # one tensor of pages with both
    c.q = torch.cat((c.q, c.q), -1)[..., :64]
    out = torch.full((64, c.heads, c.tokens), 7.0, dtype=torch.bfloat16).cuda().permute(2, 1, 0)
    wide = c.table.repeat_interleave(2, 1)
    k, v = torch.stack((c.k, c.v), 1).cuda().unbind(1)
    ws = torch.empty(32 << 20, dtype=torch.uint8).cuda()
    cabi.attention_tree(torch.cat((c.q, c.q), -1).cuda()[..., :64], k, v, wide.cuda()[:, ::2], torch.tensor([70, 300], dtype=torch.int32).cuda(),
                        c.start.cuda(), c.tree.cuda(), out, ws, 8.0)
    assert torch.equal(out, want)


def test_the_same_bits_every_time_and_in_a_graph():
    c = Case([3000, 5, 900], [4, 1, 8], 8, 2, 128, 64, torch.bfloat16, True, seed=23)
    outs = [c.call() for _ in range(3)]
    assert all(torch.equal(o, outs[0]) for o in outs[1:])
    q, k, v, table, start, tree = (x.cuda() for x in (c.q, c.k, c.v, c.table, c.start, c.tree))
    context, ws, out = torch.tensor(c.contexts, dtype=torch.int32).cuda(), torch.empty(32 << 20, dtype=torch.uint8).cuda(), torch.full_like(outs[0], 7)
    s, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=s):
        cabi.attention_tree(q, k, v, table, context, start, tree, out, ws, math.sqrt(128), stream=s.cuda_stream)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, outs[0])
    context.copy_(torch.tensor([100, 2, 4], dtype=torch.int32))  # other lengths in the same graph
    graph.replay()
    torch.cuda.synchronize()
    c.contexts = [100, 2, 4]
    assert torch.equal(out, c.call())


def test_two_streams_with_their_own_workspaces():
    cases = [Case([500, 30], [3, 2], 4, 2, 64, 16, torch.float16, True, seed=s) for s in (25, 26)]
    want = [c.call() for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    outs = [torch.full_like(w, 7) for w in want]
    spaces = [torch.empty(32 << 20, dtype=torch.uint8).cuda() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(10):
        for c, s, o, w in zip(cases, streams, outs, spaces):
            with torch.cuda.stream(s):
                c.call(out=o, workspace=w, stream=s.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, outs))


def test_empty():
    c = Case([5], [1], 2, 2, 64, 16, torch.float32, False, seed=27)
    q = torch.empty(0, 2, 64).cuda()
    cabi.attention_tree(q, c.k.cuda(), c.v.cuda(), c.table.cuda(), torch.tensor([5], dtype=torch.int32).cuda(), torch.zeros(2, dtype=torch.int32).cuda(),
                        None, q.clone(), torch.empty(32 << 20, dtype=torch.uint8).cuda(), 8.0)
