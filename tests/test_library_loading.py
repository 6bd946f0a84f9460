"""What loading the library and fa_init ask for.  No GPU needed."""
from __future__ import annotations

import os
import subprocess
import sys

import flash_attention_amd as fa

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
