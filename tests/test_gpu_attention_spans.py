"""How many tokens a launch of windowed attention is planned for: what the window
of a row tile can touch, in whole steps of 64, and not all that the sequence
holds."""
import pytest
import torch

from luisaml_amd import capi
from tests.test_gpu_attention_sinks import run

pytestmark = pytest.mark.gpu


# 512 tokens are the most that one workgroup goes through without parts
@pytest.mark.parametrize("window,n,kv", [(447, 1, 560), (447, 1, 513), (447, 1, 576), (447, 1, 577), (447, 1, 5000), (444, 4, 530)])
def test_a_window_of_eight_steps_has_no_parts(dev, window, n, kv):
    capi.kernel_trace()
    run(dev, [kv, 300], [n, 1], window, 0)
    assert "join" not in ", ".join(capi.kernel_trace())


@pytest.mark.parametrize("window,n,kv", [(448, 1, 560), (444, 5, 530), (0, 1, 560)])
def test_nine_steps_have(dev, window, n, kv):
    run(dev, [kv, 300], [n, 1], window, 0, kernel="attention_few, attention_join")


@pytest.mark.parametrize("sinks", [1, 64, 65, 200])
@pytest.mark.parametrize("over", [-1, 0, 1, 40, 64])
def test_sinks_at_the_border(dev, sinks, over):
    """Lengths about window + sinks in whole steps, of few rows and of many."""
    for n, window in ((1, 447), (90, 300)):
        run(dev, [window + n + 64 + (sinks + 63) // 64 * 64 + over], [n], window, sinks, G=4, seed=sinks + over)
    torch.cuda.synchronize()
