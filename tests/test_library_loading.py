"""What loading the library and fa_init ask for.  No GPU needed."""
from __future__ import annotations

import os
import subprocess
import sys

import flash_attention_amd as fa
from test_host_threads import compile_with_stub

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OPERATORS = ("fa_score_forward", "fa_score_backward", "fa_rotary_init", "fa_rotary", "fa_cache_append", "fa_tree_attention")


def test_a_library_without_operators_still_loads(tmp_path):
    """FA_HIP_LIBRARY may name a build from before there were operators: only their calls fail."""
    src, so = tmp_path / "old.c", tmp_path / "libold.so"
    src.write_text("".join(f"int {n}(void) {{ return 0; }}\n" for n in fa.EXPORTED_SYMBOLS if n not in OPERATORS))
    subprocess.run(["gcc", "-shared", "-fPIC", str(src), "-o", str(so)], check=True)
    code = ("import flash_attention_amd as fa\n"
            "fa.lib(); fa.init(); print('loaded')\n"
            "for call in (lambda: fa.score_attention_device(fa.score_config(0, 1, 1, 1, 8, 8, 8), 64, 64, 64, 64),\n"
            "             lambda: fa.rotary_config(0, 64)):\n"
            "    try:\n        call()\n    except fa.FaError as e:\n        print(e.status, 'no operators' in str(e))\n")
    env = dict(os.environ, FA_HIP_LIBRARY=str(so), FA_NO_TORCH_PRELOAD="1",
               PYTHONPATH=os.path.join(ROOT, "flash-attention-cpu_amd"))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, env=env, timeout=120)
    assert r.stdout.splitlines() == ["loaded", "8 True", "8 True"], (r.stdout, r.stderr)


DRIVER = r"""
int main() {
    static char mem[64] __attribute__((aligned(64)));
    void* p = mem;
    if (fa_init() != FA_OK) return 2;
    std::printf("%zu\n", stub::loaded.size());
    fa_rotary_config r;
    fa_rotary_init(&r, FA_DTYPE_F16, 64, 64, 0, 10000.0, 0, 1.0, 0.0);
    fa_rotary_tensor x{};
    x.heads = 2;
    for (int i = 0; i < 2; ++i)
        if (fa_rotary(nullptr, &r, 1, 4, static_cast<const int32_t*>(p), 0, &x, p, p, nullptr, nullptr, nullptr) != FA_OK) return 3;
    fa_score_config c{};
    c.dtype = FA_DTYPE_F16, c.batch = 1, c.heads = c.kv_heads = 2, c.seq_len_q = c.seq_len_k = 200, c.d_head = 64;
    if (fa_score_forward(nullptr, &c, p, p, p, p, nullptr) != FA_OK) return 4;
    for (const std::string& s : stub::loaded) std::printf("%s\n", s.substr(s.rfind('/') + 1).c_str());
    return 0;
}
"""


def test_operators_are_loaded_by_the_calls_that_need_them(tmp_path):
    """fa_init loads what programs without operators use, and no more."""
    exe, env = compile_with_stub(tmp_path, DRIVER)
    out = subprocess.run([exe], capture_output=True, text=True, env=env, check=True, timeout=60).stdout.split()
    assert out == ["1", "fa_kernels.hsaco", "fa_rotary.hsaco", "fa_score_f16.hsaco"]
