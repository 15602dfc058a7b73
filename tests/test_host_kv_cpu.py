"""CPU: the host driver's device caches (mh_kv_device) where the GPU refuses
memory, and in what order it sets them up, with stand-ins for the CUDA calls."""
import numpy as np
import pytest

import moe_cuda as mc
from helpers import TINY
from host_on_fake import driver, fake_library  # noqa: F401

X = np.random.default_rng(2).standard_normal((6, TINY["d_model"])).astype(np.float32)


def no_memory(f, *args):
    with pytest.raises(mc.MoeError) as e:
        f(*args)
    assert e.value.code == mc.MOE_ERR_NOMEM


@pytest.mark.parametrize("nth", range(6))
def test_a_second_call_that_finds_no_memory_leaves_the_cpu_caches(driver, nth):
    """Another type, and the n-th allocation fails: as after a first call that
    fails, the CPU's attention goes on."""
    want = driver.model(2, 12).attention(1, X, 3)
    m = driver.model(2, 12)
    m.kv_device(mc.BF16, 16)
    before = driver["live"]
    driver["fail_in"] = nth
    no_memory(m.kv_device, mc.F32, 4)
    assert before > 0 and driver["live"] == 0
    for a, b in zip(m.attention(1, X, 3), want):
        assert np.array_equal(a, b)
    m.reset()
    m.fill_kv(5, 1)
    assert m.pos() == 5


def test_device_caches_can_be_had_again_after_a_failure(driver):
    m = driver.model(2, 12)
    m.kv_device(mc.BF16, 16)
    driver["largest_ok"] = 64
    no_memory(m.kv_device, mc.F32, 16)
    driver["largest_ok"] = -1
    m.kv_device(mc.F32, 16)
    m.attention(0, X, 3)
    m.advance(3)
    m.close()
    assert driver["live"] == 0


def test_without_host_memory_either_the_calls_say_so(driver):
    m = driver.model(2, 12)
    m.kv_device(mc.F16, 16)
    driver["fail_in"] = 0
    no_memory(m.kv_device, mc.F32, 16)
    m.attention(0, X, 3)                       # sizes the step's other buffers
    m.kv_device(mc.F16, 16)
    driver["fail_in"] = 0
    no_memory(m.kv_device, mc.F32, 16)
    driver["host_limit"] = 512
    no_memory(m.attention, 0, X[:2], 1)
    no_memory(m.fill_kv, 4, 1)
    driver["host_limit"] = -1
    m.attention(0, X, 3)


def test_set_up_is_complete_before_the_caches_are_used(driver):
    """What mh_kv_device writes is read on a stream that does not wait for the
    legacy one: nothing may be left on that when the call returns."""
    m = driver.model(1, 12)
    m.kv_device(mc.F32, 16)
    assert driver["unordered"] == 0


def test_workspace_grows_in_few_steps(driver):
    """A context that grows token by token: the attention's workspace is
    allocated anew for twice the context, not for each step."""
    m = driver.model(1, 400)
    m.kv_device(mc.F32, 16)
    m.attention(0, X[:1], 1)
    driver["ws_per_kv"] = 1000
    before = driver["mallocs"]
    for _ in range(399):
        m.advance(1)
        m.attention(0, X[:1], 1)
    assert driver["short_ws"] == 0
    assert 1 <= driver["mallocs"] - before <= 9          # log2 400


def test_workspace_of_the_step_alone_where_twice_is_too_much(driver):
    m = driver.model(1, 400)
    m.kv_device(mc.F32, 16)
    m.attention(0, X[:1], 1)
    m.advance(99)
    driver["ws_per_kv"], driver["largest_ok"] = 1000, 150_000
    m.attention(0, X[:1], 1)
    assert driver["short_ws"] == 0
    m.advance(100)
    no_memory(m.attention, 0, X[:1], 1)
    driver["largest_ok"] = -1
    m.attention(0, X[:1], 1)
    assert driver["short_ws"] == 0


def test_the_type_that_is_not_named_is_the_drivers_own(driver):
    """fp32, as on the CPU: fewer bits are a caller's choice."""
    m = driver.model(1, 12)
    m.kv_device()
    m.attention(0, X[:2], 2)
    assert driver["cache_dtype"] == mc.F32
