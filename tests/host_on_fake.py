"""The C host driver compiled against fake_cuda.c: its GPU paths on the CPU."""
import ctypes as C
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
# what moe_host.c refers to and these tests do not reach
UNREACHED = ("moe_bin_close moe_bin_find moe_bin_layer_info_h moe_bin_open moe_bin_read moe_cuda_check_status moe_cuda_ep_connect "
             "moe_cuda_ep_setup moe_cuda_free_layer moe_cuda_init moe_cuda_load_bin_layer_h moe_cuda_upload_layer_dev "
             "moe_cuda_upload_layer_f32 moe_ffn moe_ffn_ep moe_quantize_rowwise_q4_dev moe_quantize_rowwise_q8_dev").split()
CUDA_HOME = os.environ.get("CUDA_HOME", "/usr/local/cuda")


def build(folder):
    """Path of the library, compiled in `folder`."""
    rest, lib = os.path.join(folder, "rest.c"), os.path.join(folder, "libmoe_host_fake.so")
    with open(rest, "w") as f:
        f.writelines(f"int {n}() {{ return 3; }}\n" for n in UNREACHED)
    inc = f"-I{CUDA_HOME}/include"
    flags = ["gcc", "-O1", "-fopenmp", "-ffp-contract=off", "-fPIC", inc]
    host, fake = os.path.join(folder, "host.o"), os.path.join(folder, "fake.o")
    subprocess.check_call(flags + ["-Dmalloc=fake_malloc", "-c", os.path.join(ROOT, "moe.cc_b200", "host", "moe_host.c"), "-o", host])
    subprocess.check_call(flags + ["-c", os.path.join(ROOT, "tests", "fake_cuda.c"), "-o", fake])
    subprocess.check_call(["gcc", "-shared", "-fopenmp", "-Wl,-Bsymbolic", "-o", lib, host, fake, rest, "-lm"])
    return lib


class Driver:
    """moe_host on the stand-ins; `models` are closed before it goes."""

    def __init__(self, mh):
        self.mh, self.lib, self.models = mh, mh.lib(), []

    def model(self, batch, max_ctx, seed=1):
        from helpers import TINY, tiny_model
        g, attn, _ = tiny_model(2, seed=seed)
        m = self.mh.HostModel(TINY, batch=batch, max_ctx=max_ctx)
        m.set_globals(g["tok_emb"], g["final_norm_w"], g["lm_head"])
        for l, a in enumerate(attn):
            m.set_layer(l, a)
        self.models.append(m)
        return m

    def __getitem__(self, name):
        return (C.c_long if name in ("largest_ok", "ws_per_kv", "host_limit") else C.c_int).in_dll(self.lib, "fake_" + name).value

    def __setitem__(self, name, v):
        (C.c_long if name in ("largest_ok", "ws_per_kv", "host_limit") else C.c_int).in_dll(self.lib, "fake_" + name).value = v


@pytest.fixture(scope="session")
def fake_library(tmp_path_factory):
    return build(str(tmp_path_factory.mktemp("fake")))


@pytest.fixture
def driver(fake_library, monkeypatch):
    import moe_host as mh
    monkeypatch.setattr(mh, "LIB_PATH", fake_library)
    monkeypatch.setattr(mh, "_lib", None)
    d = Driver(mh)
    for name, v in (("fail_in", -1), ("largest_ok", -1), ("mallocs", 0), ("live", 0), ("unordered", 0), ("ws_per_kv", 0),
                    ("short_ws", 0), ("host_limit", -1)):
        d[name] = v
    yield d
    d["host_limit"] = -1
    for m in d.models:
        m.close()
