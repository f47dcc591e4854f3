"""`import mimo_moe` with the repository's root on the path: the package itself lies in mimo-on-a-mac_b200/, whose name is
no Python name.  Importing this file puts that package in its own place in sys.modules, so there is only ever one."""
import importlib.util
import sys
from pathlib import Path

_dir = Path(__file__).resolve().parent / "mimo-on-a-mac_b200" / "mimo_moe"
_spec = importlib.util.spec_from_file_location(__name__, _dir / "__init__.py", submodule_search_locations=[str(_dir)])
sys.modules[__name__] = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(sys.modules[__name__])
