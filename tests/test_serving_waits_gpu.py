"""The bounded waits of attention by rules on tensor cores: with its loads dropped every wait runs out, the status word says so,
and the same call with the loads gives the right result afterwards.  Nothing faults or hangs."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from fluidml_b200 import cabi

DEVICE_TIMEOUT = 5


def expect_timeout_then_recover(launch, verify):
    lib = cabi.lib()
    cabi.check_device()
    try:
        cabi.check(lib.fml_debug_wait_test(2000, 1))
        launch()
        with pytest.raises(cabi.FmlError) as e:
            cabi.check_device()
        assert e.value.status == DEVICE_TIMEOUT
    finally:
        cabi.check(lib.fml_debug_wait_test(0, 0))
    cabi.check_device()
    launch()
    cabi.check_device()
    verify()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("length", [256, 700])
def test_attention_by_rules(d, length):
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(1, 4, length, d, generator=g).half().cuda() for _ in range(3))
    out, want = torch.empty_like(q), torch.empty_like(q)
    call = lambda o: cabi.attention_rules(q, k, v, o, 8.0, causal=True)  # noqa: E731
    call(want)
    expect_timeout_then_recover(lambda: call(out), lambda: None)
    assert torch.equal(out, want)


@pytest.mark.parametrize("length", [100, 1200])
def test_attention_by_rules_on_packed_pairs(length):
    """fp32 of head size 64; 1200 keys are more blocks than one accumulator takes."""
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(1, 4, length, 64, generator=g).cuda() for _ in range(3))
    out, want = torch.empty_like(q), torch.empty_like(q)
    prefix = torch.tensor([length // 3], dtype=torch.int32).cuda()
    call = lambda o: cabi.attention_rules(q, k, v, o, 8.0, cap=30.0, causal=True, prefix=prefix)  # noqa: E731
    call(want)
    expect_timeout_then_recover(lambda: call(out), lambda: None)
    assert torch.equal(out, want)
