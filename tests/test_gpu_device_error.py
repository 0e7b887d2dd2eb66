"""A device-side wait that gives up is reported, once, by the next call that looks: ``ancha_device_error``
(``fused.check_device``) for the calls that only enqueue, and every call that synchronises itself.

The wait is the self-test's, on an mbarrier that nothing arrives at, with a short budget; it ends by itself and leaves the
device usable."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from ancha_b200 import _native as N  # noqa: E402
from ancha_b200 import fused, synthetic  # noqa: E402
from ancha_b200 import microscaled as mx  # noqa: E402
from ancha_b200.model import Roformer, separate_pcm  # noqa: E402


def give_up(budget=20000):
    N.check(N.lib().ancha_wait_selftest_launch(budget, torch.cuda.current_stream().cuda_stream))


def product():
    x = torch.ones(8, 64, device="cuda")
    return mx.linear(mx.quantize(x), mx.quantize(x), dtype=torch.float32)


@pytest.mark.parametrize("budget", [0, 20000, 2000000])
def test_a_wait_that_gave_up_is_reported_once(budget):
    fused.check_device()
    give_up(budget)
    with pytest.raises(N.AnchaError, match="bounded device-side wait") as e:
        fused.check_device()
    assert e.value.status == N.E_TIMEOUT
    fused.check_device()
    assert (product() == 64).all()
    fused.check_device()


def test_enqueued_calls_neither_report_nor_clear_it():
    give_up()
    assert (product() == 64).all()  # returned before anything was known, and clears nothing
    with pytest.raises(N.AnchaError, match="bounded device-side wait"):
        fused.check_device()


def test_the_self_test_neither_takes_nor_hides_it():
    assert N.lib().ancha_wait_selftest(20000, None) == N.E_TIMEOUT
    fused.check_device()  # the self-test's own timeout is not a kernel's
    give_up()
    assert N.lib().ancha_wait_selftest(20000, None) == N.E_TIMEOUT
    with pytest.raises(N.AnchaError, match="bounded device-side wait"):
        fused.check_device()


def test_on_another_stream():
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        give_up(2000000)
        with pytest.raises(N.AnchaError, match="bounded device-side wait"):
            fused.check_device()
    fused.check_device()


def test_a_separation_reports_it(tmp_path):
    """A separation on a device where a wait gave up fails, and the next one succeeds."""
    synthetic.kernel_package(str(tmp_path), "mel-band-roformer")
    model = Roformer(str(tmp_path), 0, "f16")
    pcm = (np.sin(np.arange(9001) * 0.013) * 0.3).astype(np.float32)
    pcm = np.stack([pcm, pcm])
    want, _ = separate_pcm([model], pcm)
    give_up()
    torch.cuda.synchronize()
    with pytest.raises(N.AnchaError) as e:
        separate_pcm([model], pcm)
    assert e.value.status == N.E_TIMEOUT
    got, _ = separate_pcm([model], pcm)
    assert np.array_equal(got, want)
    model.close()


def test_budgets_outside_the_kernels_own_are_refused():
    assert N.lib().ancha_wait_selftest_launch(-1, None) == N.E_INVALID
    assert N.lib().ancha_wait_selftest_launch(1 << 40, None) == N.E_INVALID
    fused.check_device()
