"""The C host driver with its caches on the GPU (mh_kv_device) against its own
CPU attention, layer by layer on the same inputs. What a layer adds to the
residual stream may differ by the attention's rounding alone:

  fp32 cache   weights: a score errs by (head_dim + 16) 2^-23 of sum |q k| scale,
               here below 16 * 1.7^2 * 0.25 * 40 * 2^-23 < 2^-14; the CPU chain's
               own sums (up to 40 keys) stay below 2^-18. Twice that (numerator
               and sum) is below 2^-12 of max |v|.
  16-bit       q, k, v and the result are rounded by u = 2^-8 (bf16) or 2^-11
               (f16): a score errs by 2 u (1 + u) sum |q k| scale, below 24 u; the
               weights by exp of it minus 1, twice; v and the result by 2 u more.

That error of a head's output goes through |Wo|."""
import math
import os
import subprocess

import numpy as np
import pytest

from helpers import TINY, tiny_model

pytestmark = pytest.mark.gpu
mc = pytest.importorskip("moe_cuda")
mh = pytest.importorskip("moe_host")


def model(batch, max_ctx, seed=1, **variant):
    g, attn, _ = tiny_model(2, seed=seed, **variant)
    m = mh.HostModel(TINY, batch=batch, max_ctx=max_ctx)
    m.set_globals(g["tok_emb"], g["final_norm_w"], g["lm_head"])
    for l, a in enumerate(attn):
        m.set_layer(l, a)
    return m, g, attn


def head_error(dtype):
    if dtype == mc.F32:
        return 2.0**-12
    u = 2.0**-8 if dtype == mc.BF16 else 2.0**-11
    return 2 * math.expm1(24 * u) + 2.5 * u


def check_layers(host, dev, attn, ids_of_steps, dtype):
    rng = np.random.default_rng(3)
    vmax = [0.0] * TINY["n_layers"]
    for T in ids_of_steps:
        for l in range(TINY["n_layers"]):
            x = rng.standard_normal((host.batch * T, TINY["d_model"])).astype(np.float32)
            a, b = host.attention(l, x, T), dev.attention(l, x, T)
            xn = x * (1 / np.sqrt((x.astype(np.float64)**2).mean(1, keepdims=True) + 1e-6)) * attn[l]["rms1_w"]
            v = xn @ attn[l]["Wv"].T + (attn[l]["bv"] if attn[l].get("bv") is not None else 0)
            vmax[l] = max(vmax[l], float(np.abs(v).max()))
            bound = head_error(dtype) * vmax[l] * np.abs(attn[l]["Wo"]).sum(1) + 2.0**-20 * (1 + np.abs(a[0]))
            assert (np.abs(a[0] - b[0]) <= bound).all(), float((np.abs(a[0] - b[0]) / bound).max())
            assert np.isfinite(b[1]).all()
        host.advance(T)
        dev.advance(T)


@pytest.mark.parametrize("dtype", [mc.F32, mc.F16, mc.BF16])
@pytest.mark.parametrize("page,variant", [(16, {}), (1, {"qk_norm": False}), (5, {"attn_bias": True}), (64, {})])
def test_attention_matches_the_cpu_path(gpu, dtype, page, variant):
    """Prefill, single tokens and a chunk over page borders, then the same again after a reset."""
    if not variant.get("qk_norm", True) and dtype != mc.F32:
        pytest.skip("without the norm the scores of this model are unbounded: the 16-bit bound says nothing")
    host, _, attn = model(3, 40, **variant)
    dev, _, _ = model(3, 40, **variant)
    dev.kv_device(dtype, page)
    check_layers(host, dev, attn, (7, 1, 1, 20, 1, 3), dtype)
    host.reset()
    dev.reset()
    check_layers(host, dev, attn, (1, 12, 1), dtype)
    host.close()
    dev.close()


def test_a_step_that_is_taken_back(gpu):
    """Rows planned beyond what is then kept (a draft partly rejected): the next
    step's pages still hold what the kept positions were given."""
    host, _, attn = model(2, 64)
    dev, _, _ = model(2, 64)
    dev.kv_device(mc.F32, 4)
    check_layers(host, dev, attn, (10,), mc.F32)
    rng = np.random.default_rng(5)
    for l in range(TINY["n_layers"]):
        x = rng.standard_normal((2 * 14, TINY["d_model"])).astype(np.float32)
        host.attention(l, x, 14)
        dev.attention(l, x, 14)
    host.advance(6)
    dev.advance(6)
    check_layers(host, dev, attn, (9, 1), mc.F32)
    host.close()
    dev.close()


@pytest.mark.parametrize("dtype", [mc.F32, mc.BF16])
def test_filled_caches_hold_the_same_stream(gpu, dtype):
    host, _, attn = model(3, 40)
    dev, _, _ = model(3, 40)
    dev.kv_device(dtype, 16)
    for m in (host, dev):
        m.fill_kv(29, 7, 1.0)
        assert m.pos() == 29
    rng = np.random.default_rng(4)
    for l in range(TINY["n_layers"]):
        x = rng.standard_normal((3, TINY["d_model"])).astype(np.float32)
        a, b = host.attention(l, x, 1), dev.attention(l, x, 1)
        # keys and values ~ N(0, 1): |v| < 6 over these 3 * 29 * 32 numbers, sum |q k| scale < 24
        bound = head_error(dtype) * 6.0 * np.abs(attn[l]["Wo"]).sum(1) + 2.0**-20 * (1 + np.abs(a[0]))
        assert (np.abs(a[0] - b[0]) <= bound).all()
    host.close()
    dev.close()


def test_refusals(gpu):
    m, _, attn = model(1, 8)
    for args in ((2, 16), (mc.F32, 0), (7, 16)):
        with pytest.raises(mc.MoeError) as e:
            m.kv_device(*args)
        assert e.value.code == mc.MOE_ERR_INVALID
    m.kv_device(mc.F32, 16)
    m.attention(0, np.zeros((2, TINY["d_model"]), np.float32), 2)
    m.advance(2)
    with pytest.raises(mc.MoeError):
        m.kv_device(mc.F32, 16)
    with pytest.raises(mc.MoeError):                     # past max_ctx
        m.attention(0, np.zeros((7, TINY["d_model"]), np.float32), 7)
    m.close()
    odd = mh.HostModel(dict(TINY, head_dim=10), batch=1, max_ctx=8)
    with pytest.raises(mc.MoeError) as e:
        odd.kv_device(mc.F32, 16)
    assert e.value.code == mc.MOE_ERR_UNSUPPORTED
    odd.close()


def test_generation_is_repeatable_and_the_program_takes_the_option(gpu, tmp_path):
    m = mh.HostModel(TINY, batch=2, max_ctx=40, moe_base=640)
    m.kv_device(mc.BF16, 16)
    m.synth(7, 2)
    prompts = np.arange(10, dtype=np.int32).reshape(2, 5)
    a = m.generate(prompts, 20)
    assert np.array_equal(a, m.generate(prompts, 20)) and a.min() >= 0 and a.max() < TINY["vocab_size"]
    m.close()
    exe = os.path.join(os.path.dirname(mh.LIB_PATH), "moe_generate")
    r = subprocess.run([exe, "--layers", "1", "--batch", "2", "--prompt", "3", "--steps", "3", "--kv", "f32"],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and '"kv": "f32"' in r.stdout, r.stderr[-1000:]
    r = subprocess.run([exe, "--layers", "1", "--kv", "int3"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 1 and "mh_kv_device" in r.stderr
