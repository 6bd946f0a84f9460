"""The build leaves one whole set of files, and the library runs no code object of another set.  No GPU needed."""
from __future__ import annotations

import importlib.util
import os
import subprocess

import pytest

from test_host_threads import compile_with_stub

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "flash-attention-cpu_amd")


@pytest.fixture
def build(monkeypatch, tmp_path):
    spec = importlib.util.spec_from_file_location("fa_build_under_test", os.path.join(PKG, "build.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    monkeypatch.setattr(m, "HERE", str(tmp_path))
    monkeypatch.setattr(m, "LIB", str(tmp_path / "libfa_hip.so"))
    monkeypatch.setattr(m, "BUILD", str(tmp_path / "_build"))
    return m


def fake_compiler(m, monkeypatch, text, fails=""):
    """A compiler that writes `text`, after it has failed on the outputs named `fails`."""
    def run(cmd):
        out = cmd[cmd.index("-o") + 1]
        if fails and os.path.basename(out) == fails:
            raise subprocess.CalledProcessError(1, cmd)
        with open(out, "w") as f:
            f.write(text)
    monkeypatch.setattr(m, "_run", run)


@pytest.mark.parametrize("fails", ("fa_kernels.hsaco", "fa_score_bf16.hsaco", "fa_rotary.hsaco", "fa_scratch.o", "libfa_hip.so"))
def test_a_failed_build_leaves_the_last_one(build, monkeypatch, tmp_path, fails):
    fake_compiler(build, monkeypatch, "old")
    build.build()
    names = [n + ".hsaco" for n in build.OBJECTS] + ["libfa_hip.so"]
    assert all((tmp_path / n).read_text() == "old" for n in names)
    fake_compiler(build, monkeypatch, "new", fails)
    with pytest.raises(subprocess.CalledProcessError):
        build.build()
    assert {n: (tmp_path / n).read_text() for n in names} == {n: "old" for n in names}
    fake_compiler(build, monkeypatch, "new")
    build.build()
    assert all((tmp_path / n).read_text() == "new" for n in names)


def test_built_files_carry_the_stamp_of_the_present_parameters(build):
    built = [os.path.join(PKG, n + ".hsaco") for n in build.OBJECTS if n != "fa_kernels"] + [os.path.join(PKG, "libfa_hip.so")]
    for path in built:
        with open(path, "rb") as f:
            assert b"fa_ops_params_" + build.stamp().encode() in f.read(), f"{path} is of another build"


DRIVER = r"""
int main() {
    static char mem[64] __attribute__((aligned(64)));
    void* p = mem;
    stub::absent = "fa_ops_params_";
    if (fa_init() != FA_OK) return 2;
    fa_score_config c{};
    c.dtype = FA_DTYPE_BF16, c.batch = 1, c.heads = c.kv_heads = 2, c.seq_len_q = c.seq_len_k = 200, c.d_head = 64;
    fa_kv_cache k{};
    k.dtype = FA_DTYPE_F32, k.batch = 1, k.kv_heads = 2, k.d_head = 64, k.k = p, k.v = p;
    k.lens = static_cast<const int32_t*>(p), k.capacity = 50;
    fa_tree_config t{};
    t.heads = 2, t.n_tokens = 4;
    fa_append_config a{};
    a.n_tokens = 4;
    fa_rotary_config r;
    fa_rotary_init(&r, FA_DTYPE_F16, 64, 64, 0, 10000.0, 0, 1.0, 0.0);
    fa_rotary_tensor x{};
    x.heads = 2;
    float* const f = static_cast<float*>(p);
    const int32_t* const i = static_cast<const int32_t*>(p);
    std::printf("%d %d %d %d %d\n", fa_score_forward(nullptr, &c, p, p, p, p, nullptr),
                fa_score_backward(nullptr, &c, p, p, p, p, f, p, p, p, p), fa_tree_attention(nullptr, &t, &k, p, p, nullptr),
                fa_cache_append(nullptr, &k, &a, p, p, nullptr, nullptr, nullptr),
                fa_rotary(nullptr, &r, 1, 4, i, 0, &x, p, p, nullptr, nullptr, nullptr));
    std::printf("%zu\n", stub::launches.size());
    std::printf("%d\n", fa_device_v2(nullptr, f, f, f, 1, 1, 100, 100, 64, nullptr, f));
    return 0;
}
"""


def test_code_objects_of_another_build_are_refused(tmp_path):
    exe, env = compile_with_stub(tmp_path, DRIVER)
    out = subprocess.run([exe], capture_output=True, text=True, env=env, check=True, timeout=60).stdout.split("\n")
    assert out[0].split() == ["8"] * 5   # FA_ERR_MODULE
    assert out[1] == "0"                 # and nothing was launched
    assert out[2] == "0"                 # the other entry points are not concerned
