"""fml_rotary_positions against 64-bit arithmetic.

Tolerance: the functions' argument is rounded to fp32 after its reduction to half a turn (pi 2^-24 of an angle at most) and they
are good to 2 units in the last place, together 5e-7; two products and a sum in fp32 add 3 x 2^-24 of |x1| + |x2|; the result is
rounded to its type, half a step.
"""
from fractions import Fraction

import pytest
import torch

pytestmark = pytest.mark.gpu

from fluidml_b200 import cabi
from serving_oracle import HALF_STEP, TYPES

FREQ = {n: torch.tensor([10000.0 ** (-i / n) for i in range(n)], dtype=torch.float32) for n in (1, 2, 4, 5, 8, 10, 16, 32, 40, 64)}


TURN = Fraction("6.28318530717958647692528676655900576839433879875021")


def reduced(position, frequency):
    """position * frequency less whole turns, exact but for the last rounding."""
    angle = position * Fraction(frequency)
    return float(angle - round(angle / TURN) * TURN)


def oracle(x, positions, f, magnitude, interleaved):
    """(turned x in 64 bits, |x1| + |x2| of every feature's pair)"""
    x = x.double().cpu()
    n = len(f)
    angle = torch.tensor([[reduced(int(p), float(w)) for w in f] for p in positions], dtype=torch.float64).reshape(-1, n)
    c, s = (torch.cos(angle) * magnitude)[:, None], (torch.sin(angle) * magnitude)[:, None]
    first = torch.arange(n) * 2 if interleaved else torch.arange(n)
    second = first + (1 if interleaved else n)
    y, size = x.clone(), torch.zeros_like(x)
    y[..., first], y[..., second] = x[..., first] * c - x[..., second] * s, x[..., second] * c + x[..., first] * s
    size[..., first] = size[..., second] = (x[..., first].abs() + x[..., second].abs()) * magnitude
    return y, size


def hold(got, want, size):
    err = (got.double().cpu() - want).abs()
    assert (err <= 1e-6 * size + HALF_STEP[got.dtype] * want.abs() + 1e-30).all(), float(err.max())


def randn(seed, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("layout", [cabi.ROTARY_HALVES, cabi.ROTARY_INTERLEAVED])
@pytest.mark.parametrize("heads,kv,head,pairs", [(4, 2, 64, 8), (3, 3, 64, 32), (8, 1, 128, 64), (2, 2, 80, 40), (2, 1, 80, 10), (5, 1, 6, 1), (1, 1, 20, 5)])
def test_shapes_and_types(dtype, layout, heads, kv, head, pairs):
    t, n = TYPES[dtype], 37
    q, k, v = randn(1, n, heads, head, dtype=t), randn(2, n, kv, head, dtype=t), randn(3, n, kv, head, dtype=t)
    positions = torch.randint(0, 1 << 20, (n,), generator=torch.Generator().manual_seed(4))
    f = FREQ[pairs] if pairs in FREQ else FREQ[64][:pairs]
    qo, ko, vo = torch.full_like(q, 7), torch.full_like(k, 7), torch.full_like(v, 7)
    cabi.rotary_positions(q, k, v, positions.cuda(), None, f.cuda(), qo, ko, vo, magnitude=1.25, layout=layout)
    for x, y in ((q, qo), (k, ko)):
        hold(y, *oracle(x, positions, f, 1.25, layout == cabi.ROTARY_INTERLEAVED))
        assert torch.equal(y[..., 2 * pairs:], x[..., 2 * pairs:])
    assert torch.equal(vo, v)
    cabi.check_device()


@pytest.mark.parametrize("tokens", [1, 2, 255, 1031])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_append_to_a_paged_cache(tokens, dtype):
    t, kv, head, page = TYPES[dtype], 2, 64, 24
    src = randn(5, tokens, (3 + 2 * kv) * head, dtype=t)  # one projection: strided views
    q, k, v = (x.unflatten(-1, (-1, head)) for x in src.split((3 * head, kv * head, kv * head), -1))
    pages = -(-tokens // page) + 2
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(6))[:tokens].to(torch.int32)
    slots[tokens // 2] = -1  # padding: left out
    positions = torch.arange(tokens, dtype=torch.int32) + 100
    kc, vc, qo = (torch.full((pages, page, kv, head), 3.0, dtype=t).cuda() for _ in range(2)).__iter__(), None, torch.empty(tokens, 3, head, dtype=t).cuda()
    kc, vc = kc
    cabi.rotary_positions(q, k, v, positions.cuda(), slots.cuda(), FREQ[16].cuda(), qo, kc, vc)
    cabi.check_device()
    want, size = oracle(k, positions, FREQ[16], 1.0, False)
    k_flat, v_flat = kc.flatten(0, 1).cpu(), vc.flatten(0, 1).cpu()
    kept = slots >= 0
    hold(k_flat[slots[kept].long()], want[kept], size[kept])
    assert torch.equal(v_flat[slots[kept].long()], v.cpu()[kept])
    rest = torch.ones(pages * page, dtype=torch.bool)
    rest[slots[kept].long()] = False
    assert (k_flat[rest] == 3).all() and (v_flat[rest] == 3).all()
    hold(qo, *oracle(q, positions, FREQ[16], 1.0, False))


def test_slots_beyond_the_cache_are_left_out_and_recorded():
    k, kc = randn(1, 3, 1, 8), torch.zeros(2, 4, 1, 8).cuda()
    cabi.rotary_positions(None, k, None, torch.arange(3).cuda(), torch.tensor([8, 2, 1 << 40]).cuda(), FREQ[4].cuda(), None, kc, None)
    with pytest.raises(cabi.FmlError) as e:
        cabi.check_device()
    assert e.value.status == 7
    assert (kc.flatten(0, 1)[[0, 1, 3, 4, 5, 6, 7]] == 0).all() and (kc[0, 2] != 0).any()
    cabi.check_device()


def test_in_place_and_values_alone():
    x = randn(9, 50, 4, 64, dtype=torch.bfloat16)
    y, p = x.clone(), torch.arange(50).cuda()
    cabi.rotary_positions(y, None, None, p, None, FREQ[32].cuda(), y, None, None)
    hold(y, *oracle(x, p, FREQ[32], 1.0, False))
    vc = torch.zeros(4, 16, 4, 64, dtype=torch.bfloat16).cuda()
    cabi.rotary_positions(None, None, x, p, p, torch.empty(0).cuda(), None, None, vc)
    assert torch.equal(vc.flatten(0, 1)[:50], x)


def test_strides_alignment_and_empty():
    base = randn(11, 9, 5, 65)
    for x in (base[..., 1:], base[:, ::2, :64], base.transpose(0, 1)[..., :64], base[:, :, :64].flip(0)):
        n = x.shape[0]
        out = torch.empty(64, x.shape[1], n).cuda().permute(2, 1, 0)  # features outermost
        for layout in (0, 1):
            cabi.rotary_positions(x, None, None, torch.arange(n).cuda() * 1000, None, FREQ[8].cuda(), out, None, None, layout=layout)
            hold(out, *oracle(x, torch.arange(n) * 1000, FREQ[8], 1.0, layout == 1))
    empty = torch.empty(0, 2, 64).cuda()
    cabi.rotary_positions(empty, None, None, torch.empty(0, dtype=torch.int64).cuda(), None, FREQ[8].cuda(), empty.clone(), None, None)


def test_far_and_negative_positions():
    x = randn(12, 4, 1, 128)
    p = torch.tensor([-5, (1 << 31) + 7, 1 << 36, 16777217])
    out = torch.empty_like(x)
    cabi.rotary_positions(x, None, None, p.cuda(), None, FREQ[64].cuda(), out, None, None)
    hold(out, *oracle(x, p, FREQ[64], 1.0, False))


def test_positions_beyond_what_a_double_holds():
    p = torch.tensor([1 << 53, (1 << 53) + 1, -(1 << 53) - 1, (1 << 57) + 2047, (1 << 60) + 1, (1 << 62) + 12345, (1 << 63) - 1, -(1 << 63), 1 - (1 << 63)])
    x = randn(14, len(p), 1, 128)
    out = torch.empty_like(x)
    cabi.rotary_positions(x, None, None, p.cuda(), None, FREQ[64].cuda(), out, None, None)
    hold(out, *oracle(x, p, FREQ[64], 1.0, False))


def test_a_stream_of_its_own_and_a_captured_graph():
    x, p, f = randn(13, 8, 2, 64), torch.arange(8).cuda(), FREQ[16].cuda()
    out = torch.zeros_like(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        cabi.rotary_positions(x, None, None, p, None, f, out, None, None, stream=s.cuda_stream)
    p += 11
    graph.replay()
    torch.cuda.synchronize()
    hold(out, *oracle(x, torch.arange(8) + 11, FREQ[16], 1.0, False))
