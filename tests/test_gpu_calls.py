"""GPU: the Python calls of a decode step through ctypes, where the extension was
not built: the tests of the calls themselves, taken that way."""
import pytest

import moe_cuda as mc
import test_gpu_attn as ta
import test_gpu_route as tr
from test_calls_cpu import without_extension  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def test_calls_through_ctypes(gpu, without_extension):  # noqa: F811
    ta.test_a_step_written_just_before_it_is_read(gpu)
    ta.test_plan_limits(gpu)
    ta.test_attention_layout_strides_and_bad_pages(gpu, torch.bfloat16, 24)
    ta.test_attention_in_place_repeatable_and_on_another_stream(gpu)
    ta.test_norm_rope_append(gpu, torch.float32, torch.bfloat16, 8, 2, 256, 64, 24, 7, True)
    ta.test_norm_rope_append(gpu, torch.float16, torch.float16, 7, 1, 80, 40, 5, 3, True)
    tr.test_route(gpu, torch.float32, "sigmoid", 33, 256, 8, 8, 4, 2, True, True)
    tr.test_strided_rows_another_stream_and_repeat(gpu)
    assert mc.route.__module__ == "moe_calls"
