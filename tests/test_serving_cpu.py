"""Arguments that the serving operators refuse, and their host computations: no device needed."""
import ctypes
import math
import os
import subprocess
import sysconfig

import numpy as np
import pytest
import torch

from fluidml_b200 import cabi

BAD_ARG, UNSUPPORTED, MISALIGNED = 1, 2, 3


def described(shape, dtype=cabi.F32, strides=None, data=1 << 20):
    """A description without memory behind it: every call below is refused before any of it is touched."""
    t = cabi.Tensor()
    t.data, t.dtype, t.rank = data, dtype, len(shape)
    for i, (n, s) in enumerate(zip(shape, strides or cabi.gen_strides(shape))):
        t.shape[i], t.stride[i] = n, s
    return t


def refused(status, call, *args, **kw):
    with pytest.raises(cabi.FmlError) as e:
        call(*args, **kw)
    assert e.value.status == status, str(e.value)


# ------------------------------------------------------------------ rotary positions
def rotary(**kw):
    a = dict(q=described((5, 4, 64)), k=described((5, 2, 64)), v=described((5, 2, 64)), positions=described((5,), cabi.I64), slots=None,
             frequencies=described((16,)), q_out=described((5, 4, 64)), k_out=described((5, 2, 64)), v_out=described((5, 2, 64)))
    a.update(kw)
    return a


PAGED = dict(slots=described((5,), cabi.I32), k_out=described((3, 4, 2, 64)), v_out=described((3, 4, 2, 64)))


@pytest.mark.parametrize("kw", [
    dict(q=None, k=None, v=None, q_out=None, k_out=None, v_out=None),
    dict(q_out=None), dict(k=None), dict(layout=2), dict(magnitude=math.nan),
    dict(positions=described((4,), cabi.I64)), dict(positions=described((5,), cabi.F32)), dict(positions=described((5,), cabi.I64, data=None)),
    dict(frequencies=described((33,))), dict(frequencies=described((16,), cabi.F16)), dict(frequencies=described((16, 1))),
    dict(q=described((5, 4, 64), cabi.F16)), dict(q=described((5, 4, 64), cabi.I32)), dict(q=described((5, 256))),
    dict(k=described((6, 2, 64))), dict(k=described((5, 2, 32))), dict(k_out=described((5, 3, 64))), dict(v_out=described((5, 2, 64), cabi.BF16)),
    dict(slots=described((5,), cabi.I32)),  # caches of rank 3
    dict(PAGED, slots=described((6,), cabi.I32)), dict(PAGED, slots=described((5,), cabi.BOOL)), dict(PAGED, k_out=described((3, 4, 1, 64))),
    dict(PAGED, v_out=described((4, 4, 2, 64))), dict(PAGED, v_out=described((4, 3, 2, 64))),
    dict(q_out=described((5, 4, 64), strides=[64, 320, 1])),  # in place with other strides
    dict(q=described((5, 4, -1)), q_out=described((5, 4, -1))),
])
def test_rotary_refusals(kw):
    refused(BAD_ARG, cabi.rotary_positions, **rotary(**kw))


def test_rotary_slots_need_keys_or_values():
    refused(BAD_ARG, cabi.rotary_positions, **rotary(k=None, v=None, k_out=None, v_out=None, slots=described((5,), cabi.I32)))


@pytest.mark.parametrize("heads,head", [(1, 1 << 34), ((1 << 20) - 1, 1 << 15), (1 << 16, 1 << 15)])
def test_rotary_features_beyond_32_bits(heads, head):
    x = described((1, heads, head), cabi.F16)
    refused(UNSUPPORTED, cabi.rotary_positions, **rotary(q=x, q_out=x, k=None, k_out=None, v=None, v_out=None, positions=described((1,), cabi.I64)))


def test_frequencies_of_every_scaling():
    rot, base, factor, length = 64, 10000.0, 8.0, 4096.0
    i = np.arange(rot // 2)
    plain = base ** (-2.0 * i / rot)
    got, magnitude = cabi.rotary_frequencies(rot)
    np.testing.assert_allclose(got, plain, rtol=2 ** -24 * 1.01)
    assert magnitude == 1.0
    got, _ = cabi.rotary_frequencies(rot, cabi.ROTARY_LINEAR, factor=factor)
    np.testing.assert_allclose(got, plain / factor, rtol=2 ** -24 * 1.01)
    got, _ = cabi.rotary_frequencies(rot, cabi.ROTARY_NTK, factor=factor)
    np.testing.assert_allclose(got, (base * factor ** (rot / (rot - 2))) ** (-2.0 * i / rot), rtol=2 ** -24 * 1.01)
    got, _ = cabi.rotary_frequencies(rot, cabi.ROTARY_BANDS, factor=factor, trained_length=length, turns_low=1, turns_high=4)
    turns = length * plain / (2 * math.pi)
    want = np.where(turns >= 4, plain, np.where(turns <= 1, plain / factor, plain * ((turns - 1) / 3 + (1 - (turns - 1) / 3) / factor)))
    np.testing.assert_allclose(got, want, rtol=2 ** -24 * 1.01)
    got, magnitude = cabi.rotary_frequencies(rot, cabi.ROTARY_RAMP, factor=factor, trained_length=length, turns_low=1, turns_high=32)
    pair = lambda n: rot * math.log(length / (n * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
    lo, hi = math.floor(pair(32)), math.ceil(pair(1))
    assert 0 < lo < hi < rot // 2
    stretch = np.clip((i - lo) / (hi - lo), 0, 1)
    np.testing.assert_allclose(got, plain / factor * stretch + plain * (1 - stretch), rtol=2 ** -24 * 1.01)
    assert magnitude == pytest.approx(0.1 * math.log(factor) + 1, rel=2 ** -23)
    assert cabi.rotary_frequencies(2)[0].tolist() == [1.0]


@pytest.mark.parametrize("kw", [dict(rot=0), dict(rot=7), dict(rot=64, base=1.0), dict(rot=64, base=math.inf), dict(rot=64, scaling=5),
                                dict(rot=64, scaling=cabi.ROTARY_LINEAR, factor=0.5), dict(rot=2, scaling=cabi.ROTARY_NTK, factor=2.0),
                                dict(rot=64, scaling=cabi.ROTARY_BANDS, factor=2.0), dict(rot=64, scaling=cabi.ROTARY_RAMP, factor=2.0,
                                                                                          trained_length=100.0, turns_low=4.0, turns_high=4.0)])
def test_frequency_refusals(kw):
    refused(BAD_ARG, cabi.rotary_frequencies, **kw)


# ------------------------------------------------------------------ attention by rules
def rules(**kw):
    a = dict(q=described((2, 4, 7, 64)), k=described((2, 2, 9, 64)), v=described((2, 2, 9, 64)), out=described((2, 4, 7, 64)), divisor=8.0)
    a.update(kw)
    return a


@pytest.mark.parametrize("status,kw", [
    (BAD_ARG, dict(divisor=0.0)), (BAD_ARG, dict(divisor=math.inf)), (BAD_ARG, dict(cap=-1.0)), (BAD_ARG, dict(cap=math.nan)),
    (BAD_ARG, dict(q=described((4, 7, 64)))), (BAD_ARG, dict(q=None)), (BAD_ARG, dict(out=described((2, 4, 9, 64)))),
    (BAD_ARG, dict(v=described((2, 2, 8, 64)))), (BAD_ARG, dict(k=described((1, 2, 9, 64)), v=described((1, 2, 9, 64)))),
    (BAD_ARG, dict(k=described((2, 3, 9, 64)), v=described((2, 3, 9, 64)))), (BAD_ARG, dict(k=described((2, 0, 9, 64)), v=described((2, 0, 9, 64)))),
    (BAD_ARG, dict(out=described((2, 4, 7, 64), cabi.F16))), (BAD_ARG, dict(slopes=described((2,)))), (BAD_ARG, dict(slopes=described((4,), cabi.BF16))),
    (BAD_ARG, dict(prefix=described((3,), cabi.I32))), (BAD_ARG, dict(prefix=described((2,)))),
    (BAD_ARG, dict(q_documents=described((2, 7), cabi.I32))), (BAD_ARG, dict(k_documents=described((2, 9), cabi.I32))),
    (BAD_ARG, dict(q_documents=described((2, 7), cabi.I32), k_documents=described((2, 7), cabi.I32))),
    (UNSUPPORTED, dict(q=described((2, 4, 7, 132)), k=described((2, 2, 9, 132)), v=described((2, 2, 9, 132)), out=described((2, 4, 7, 132)))),
    (UNSUPPORTED, dict(q=described((2, 4, 7, 6)), k=described((2, 2, 9, 6)), v=described((2, 2, 9, 6)), out=described((2, 4, 7, 6)))),
])
def test_rules_refusals(status, kw):
    refused(status, cabi.attention_rules, **rules(**kw))


# ------------------------------------------------------------------ attention of a tree
class Bytes:
    """Stands for device memory that is never reached."""
    def __init__(self, place, size):
        self.place, self.size = place, size

    def data_ptr(self):
        return self.place

    def numel(self):
        return self.size

    def element_size(self):
        return 1


def tree(**kw):
    a = dict(q=described((6, 4, 64)), k_cache=described((9, 16, 2, 64)), v_cache=described((9, 16, 2, 64)),
             block_table=described((2, 3), cabi.I32), context=described((2,), cabi.I32), query_start=described((3,), cabi.I32),
             tree=described((6,), cabi.I64), out=described((6, 4, 64)), workspace=Bytes(1 << 20, 64 << 20), divisor=8.0)
    a.update(kw)
    return a


@pytest.mark.parametrize("status,kw", [
    (BAD_ARG, dict(divisor=0.0)), (BAD_ARG, dict(cap=math.inf)), (BAD_ARG, dict(q=described((6, 5, 64)), out=described((6, 5, 64)))),
    (BAD_ARG, dict(out=described((6, 4, 32)))), (BAD_ARG, dict(v_cache=described((8, 16, 2, 64)))),
    (BAD_ARG, dict(k_cache=described((9, 16, 2, 64), cabi.F16))), (BAD_ARG, dict(k_cache=described((9, 0, 2, 64)), v_cache=described((9, 0, 2, 64)))),
    (BAD_ARG, dict(block_table=described((2, 3), cabi.I64))), (BAD_ARG, dict(block_table=described((2,), cabi.I32))),
    (BAD_ARG, dict(context=described((3,), cabi.I32))), (BAD_ARG, dict(context=described((2,), cabi.I64))),
    (BAD_ARG, dict(query_start=described((2,), cabi.I32))), (BAD_ARG, dict(tree=described((6,), cabi.I32))), (BAD_ARG, dict(tree=described((5,), cabi.I64))),
    (BAD_ARG, dict(slopes=described((2,)))), (BAD_ARG, dict(workspace=Bytes(1 << 20, 1000))), (BAD_ARG, dict(workspace=Bytes((1 << 20) + 8, 64 << 20))),
    (UNSUPPORTED, dict(q=described((6, 4, 66)), out=described((6, 4, 66)), k_cache=described((9, 16, 2, 66)), v_cache=described((9, 16, 2, 66)))),
    (UNSUPPORTED, dict(q=described((6, 4, 132)), out=described((6, 4, 132)), k_cache=described((9, 16, 2, 132)), v_cache=described((9, 16, 2, 132)))),
    (MISALIGNED, dict(k_cache=described((9, 16, 2, 64), data=(1 << 20) + 4))), (MISALIGNED, dict(v_cache=described((9, 16, 2, 64), strides=[4096, 256, 65, 1]))),
    (MISALIGNED, dict(v_cache=described((9, 16, 2, 64), strides=[2048, 128, 1, 2]))),
])
def test_tree_refusals(status, kw):
    refused(status, cabi.attention_tree, **tree(**kw))


def test_tree_rows_next_to_what_32_bits_count():
    tokens, heads = 151 * 331, 2 * 9 * 7 * 11 * 31  # 2^31 - 2 rows of one kv head, in tiles that end behind 2^31
    refused(UNSUPPORTED, cabi.attention_tree, **tree(q=described((tokens, heads, 8), cabi.F16), out=described((tokens, heads, 8), cabi.F16), tree=None,
                                                     k_cache=described((9, 16, 1, 8), cabi.F16), v_cache=described((9, 16, 1, 8), cabi.F16)))


@pytest.mark.parametrize("kw", [dict(cap=1e30), dict(cap=3e38), dict(cap=1e-30), dict(divisor=1e-39), dict(divisor=-1e-40), dict(divisor=3e38),
                                dict(divisor=1e25, cap=1e18), dict(divisor=1e-25, cap=1e-18)])
def test_factors_beyond_fp32(kw):
    refused(UNSUPPORTED, cabi.attention_rules, **rules(**kw))
    refused(UNSUPPORTED, cabi.attention_tree, **tree(**kw))


def test_tree_workspace_sizes():
    assert cabi.attention_tree_workspace(1, 1, 8, 3, 64) == 0 and cabi.attention_tree_workspace(1, 1, 8, 8, 129) == 0
    small, large = cabi.attention_tree_workspace(4, 4, 8, 2, 64), cabi.attention_tree_workspace(4, 400, 8, 2, 128)
    assert 0 < small < large < 32 << 20


@pytest.mark.parametrize("heads,kv,d", [(32, 8, 128), (16, 16, 64), (8, 1, 128), (4, 4, 32)])
def test_a_workspace_for_many_requests_is_enough_for_fewer(heads, kv, d):
    """The need of a call follows the rows that a request has on average, so it rises as requests fall; the query does not."""
    def taken(requests, tokens, size):
        """Whether a call takes a workspace of `size` bytes; without a device every call ends at the outputs' check, which follows."""
        with pytest.raises(cabi.FmlError) as e:
            cabi.attention_tree(**tree(q=described((tokens, heads, d)), out=described((tokens, heads, d)), k_cache=described((9, 16, kv, d)),
                                       v_cache=described((9, 16, kv, d)), block_table=described((requests, 3), cabi.I32),
                                       context=described((requests,), cabi.I32), query_start=described((requests + 1,), cabi.I32), tree=None,
                                       workspace=Bytes(1 << 20, size)))
        return "workspace of" not in str(e.value)

    for requests, tokens in ((64, 64), (1, 1), (3, 64), (200, 1000)):
        size = cabi.attention_tree_workspace(requests, tokens, heads, kv, d)
        for fewer in {1, min(2, requests), requests // 8, requests // 2, requests} - {0}:
            for t in {1, tokens // 3, tokens} - {0}:
                assert taken(fewer, t, size), (requests, tokens, fewer, t)
                assert cabi.attention_tree_workspace(fewer, t, heads, kv, d) <= size
        assert not taken(requests, tokens, 4096)


# ------------------------------------------------------------------ sampling
def sampling(**kw):
    a = dict(logits=described((3, 100)), uniform=described((3,)), tokens=described((3,), cabi.I64))
    a.update(kw)
    return a


@pytest.mark.parametrize("status,kw", [
    (BAD_ARG, dict(logits=described((3, 100), cabi.I32))), (BAD_ARG, dict(logits=described((100,)))), (BAD_ARG, dict(uniform=described((4,)))),
    (BAD_ARG, dict(uniform=described((3,), cabi.F16))), (BAD_ARG, dict(uniform=None)), (BAD_ARG, dict(tokens=None)),
    (BAD_ARG, dict(tokens=described((3,)))), (BAD_ARG, dict(temperature=described((1,)))), (BAD_ARG, dict(top_k=described((3,)))),
    (BAD_ARG, dict(top_p=described((3,), cabi.I32))), (BAD_ARG, dict(min_p=described((2,)))), (BAD_ARG, dict(probabilities=described((3,), cabi.BF16))),
    (UNSUPPORTED, dict(logits=described((3, (1 << 18) + 1)))), (UNSUPPORTED, dict(logits=described((3, 0)))),
])
def test_sample_refusals(status, kw):
    refused(status, cabi.sample, **sampling(**kw))


# ------------------------------------------------------------------ the extension behind the calls
def test_everything_else_builds_without_the_headers_of_python(monkeypatch, tmp_path):
    import fluidml_b200.build as b
    built = []
    for name in ("build_kernels", "build_host", "build_cli"):
        monkeypatch.setattr(b, name, lambda verbose=False, name=name: built.append(name))
    monkeypatch.setattr(b, "SERVING_SO", str(tmp_path / os.path.basename(b.SERVING_SO)))
    monkeypatch.setattr(b.sysconfig, "get_paths", lambda: {"include": str(tmp_path)})
    b.build_all()
    assert built == ["build_kernels", "build_host", "build_cli"] and not os.path.exists(b.SERVING_SO)


def test_the_extension_is_this_interpreters():
    """Another version of Python has another layout of its objects: it must not load what was built for this one."""
    import fluidml_b200.build as b
    assert os.path.basename(b.SERVING_SO) == "_serving" + sysconfig.get_config_var("EXT_SUFFIX")
    with pytest.raises(cabi.FmlError):
        cabi.sample(**sampling(uniform=None))  # loads it
    assert os.path.realpath(cabi._native.__file__) == os.path.realpath(b.SERVING_SO)


# ------------------------------------------------------------------ where tensors are
@pytest.mark.parametrize("call,args", [
    (cabi.rotary_positions, rotary(q_out=described((5, 4, 64), strides=[64, 0, 1]))),
    (cabi.rotary_positions, rotary(**dict(PAGED, k_out=described((3, 4, 2, 64), data=2 << 20),
                                        v_out=described((3, 4, 2, 64), strides=[0, 128, 64, 1], data=3 << 20)))),
    (cabi.attention_rules, rules(out=described((2, 4, 7, 64), strides=[0, 448, 64, 1]))),
    (cabi.attention_tree, tree(out=described((6, 4, 64), strides=[256, 64, 0]))),
    (cabi.sample, sampling(tokens=described((3,), cabi.I64, strides=[0]))),
    (cabi.sample, sampling(probabilities=described((3,), strides=[0]))),
])
def test_outputs_whose_elements_share_a_place_are_refused(call, args):
    with pytest.raises(cabi.FmlError) as e:
        call(**args)
    assert e.value.status == BAD_ARG and "stride of 0" in str(e.value)


@pytest.mark.skipif(torch.cuda.device_count() == 1, reason="with one device its memory is the only one there is")
@pytest.mark.parametrize("call,args", [(cabi.rotary_positions, rotary()), (cabi.attention_rules, rules()), (cabi.attention_tree, tree()),
                                       (cabi.sample, sampling())])
def test_inputs_elsewhere_are_refused(call, args):
    """The descriptions' memory is no device's: a launch on it would fault."""
    with pytest.raises(cabi.FmlError) as e:
        call(**args)
    assert e.value.status == BAD_ARG and "an input is not memory of the current device" in str(e.value)


def test_structures_are_the_headers(tmp_path):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    source = tmp_path / "sizes.c"
    source.write_text('#include <stdio.h>\n#include "fluidml_cuda.h"\nint main(void) { printf("%zu %zu %d %d %d %d", sizeof(fml_rotary_spec), '
                      'sizeof(fml_score_rules), FML_F16, FML_BF16, FML_ROTARY_RAMP, FML_ROTARY_INTERLEAVED); return 0; }\n')
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(source), "-o", str(tmp_path / "sizes")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "sizes")], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(cabi.RotarySpec), ctypes.sizeof(cabi.ScoreRules), cabi.F16, cabi.BF16, cabi.ROTARY_RAMP, cabi.ROTARY_INTERLEAVED]


def test_other_operators_refuse_the_types_they_do_not_take():
    a, b, c = (described((4, 8), cabi.F16) for _ in range(3))
    for call in (lambda: cabi.copy_strided(_Held(a), _Held(b)), lambda: cabi.elementwise(cabi.ADD, _Held(a), _Held(b), _Held(c)),
                 lambda: cabi.softmax(_Held(a), None, 1.0, _Held(b), 1)):
        with pytest.raises(cabi.FmlError):
            call()


class _Held:
    def __init__(self, t):
        self.t = t

    def c(self):
        return self.t
