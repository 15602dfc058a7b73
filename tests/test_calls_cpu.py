"""CPU: the Python calls of a decode step where the CPython extension was not
built: there, and refusing what the extension refuses."""
import inspect

import pytest

import moe_cuda as mc
import test_attn_cpu

NAMES = ("kv_plan", "qk_norm_rope", "paged_attention", "route")
torch = pytest.importorskip("torch")


@pytest.fixture
def without_extension(monkeypatch, tmp_path):
    for n in NAMES:
        monkeypatch.delattr(mc, n, raising=False)
    monkeypatch.setattr(mc, "FAST_PATH", str(tmp_path / "_moe_fast.so"))
    yield mc
    for n in NAMES:
        mc.__dict__.pop(n, None)


def test_the_calls_are_there(without_extension):
    for n in NAMES:
        assert inspect.isfunction(getattr(mc, n)) and getattr(mc, n).__module__ == "moe_calls"
    test_attn_cpu.test_binding_arguments()
    test_attn_cpu.test_binding_refuses_host_tensors_and_wrong_types()


def test_both_forms_take_the_same_arguments():
    import moe_calls
    for n in NAMES:
        documented = {}
        exec("def " + getattr(mc, n).__doc__.split("\n\n")[0] + ": pass", documented)
        assert inspect.signature(documented[n]) == inspect.signature(getattr(moe_calls, n))


def test_arguments_that_are_not_what_they_should_be(without_extension):
    x, i, p = torch.zeros(2, 8), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, 2)
    for f in (lambda: mc.route(x, i, p, score="tanh"), lambda: mc.kv_plan(i, i, "16", 2, i, i, i, i, i),
              lambda: mc.paged_attention(x, x, x, i, i, x, None, 16, 1.0), lambda: mc.paged_attention(None, None, None, i, i, x, None, 16, 1.0),
              lambda: mc.qk_norm_rope(x, x, x, x, None, i, i, x)):
        with pytest.raises(mc.MoeError) as e:
            f()
        assert e.value.code == mc.MOE_ERR_INVALID
