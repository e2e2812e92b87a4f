"""The package is found with only the repository's root on the path."""

import os
import shutil
import subprocess
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]


def _python(code, cwd):
    env = {k: v for k, v in os.environ.items() if k != "PYTHONPATH"}
    return subprocess.run([sys.executable, "-c", code], cwd=cwd, env=env, capture_output=True, text=True)


def test_import_from_the_repositorys_root(tmp_path):
    code = ("import breeze_b200, sys\nfrom breeze_b200.fused import paged\nfrom breeze_b200 import _lib\n"
            "assert paged._lib is _lib and sys.modules['breeze_b200'] is breeze_b200 and breeze_b200.__version__\n"
            "print(breeze_b200.__file__, _lib.LIB_PATH.parent)\n")
    home = ROOT / "breeze-tts-2_b200" / "breeze_b200"
    for cwd, first in ((ROOT, ""), (tmp_path, f"import sys; sys.path.insert(0, {str(ROOT)!r})\n")):
        r = _python(first + code, cwd)
        assert r.returncode == 0, r.stderr
        assert r.stdout.split() == [str(home / "__init__.py"), str(home)]


def test_the_case_file_finds_the_package_wherever_it_lies(tmp_path):
    """Its own calls get as far as the operators' refusal of CPU tensors."""
    shutil.copy(ROOT / "perf" / "operators.py", tmp_path / "cases.py")
    code = f"""
import sys
sys.path[:0] = [{str(ROOT)!r}, {str(tmp_path)!r}]
import cases, torch
cases.own = True
for op in ("append", "paged"):
    case = dict(op=op, heads=1, kv_heads=1)
    row = torch.zeros(1, 192, dtype=torch.bfloat16)
    pages = torch.zeros(1, 1, 16, 64, dtype=torch.bfloat16)
    state = dict(case=case, k_pages=pages, v_pages=pages, page_table=torch.zeros(1, 1, dtype=torch.int32),
                 seq_lens=torch.ones(1, dtype=torch.int32), q_starts=None, max_q=1, qkv=row, q=row[:, :64],
                 cos=torch.ones(1, 64), sin=torch.ones(1, 64), q_norm=None, k_norm=None)
    try:
        cases.run(state)
    except RuntimeError as e:
        assert "CUDA tensors" in str(e), e
    else:
        raise AssertionError("CPU tensors were taken")
"""
    r = _python(code, ROOT)
    assert r.returncode == 0, r.stderr
