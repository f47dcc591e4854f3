"""The package is importable with the repository's root on the path, as with its own folder, and is the same package."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
PACKAGE = ROOT / "mimo-on-a-mac_b200"


def run(code, cwd, *paths):
    """`code` in a Python of its own that has `paths` first on its path and nothing of this repository else."""
    head = f"import sys; sys.path[:0] = {[str(p) for p in paths]!r}; "
    env = {k: v for k, v in os.environ.items() if k != "PYTHONPATH"}
    return subprocess.run([sys.executable, "-c", head + code], cwd=cwd, env=env, capture_output=True, text=True)


FORMS = ["from mimo_moe import paged", "import mimo_moe.paged", "import mimo_moe",
         "from mimo_moe.layer import AttentionConfig"]


@pytest.mark.parametrize("paths,first", [((ROOT,), f) for f in FORMS] + [((PACKAGE,), FORMS[0]),
                         ((ROOT, PACKAGE), FORMS[0]), ((PACKAGE, ROOT), FORMS[0])])
def test_package_from_each_folder(tmp_path, paths, first):
    code = (f"{first}; import mimo_moe, mimo_moe.paged, mimo_moe.layer; from mimo_moe import paged, layer; "
            "assert sys.modules['mimo_moe'] is mimo_moe and mimo_moe.paged is paged; "
            "assert paged.AttentionConfig is layer.AttentionConfig; print(mimo_moe.__file__, paged.__file__)")
    done = run(code, tmp_path, *paths)
    assert done.returncode == 0, done.stderr
    folder = PACKAGE / "mimo_moe"
    assert done.stdout.split() == [str(folder / "__init__.py"), str(folder / "paged.py")]
