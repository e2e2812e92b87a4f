"""``import breeze_b200`` with this directory on sys.path: the package of that
name in breeze-tts-2_b200/ takes this module's place."""

import importlib.util
import sys
from pathlib import Path

_package = Path(__file__).resolve().parent / "breeze-tts-2_b200" / "breeze_b200"
_spec = importlib.util.spec_from_file_location(__name__, _package / "__init__.py", submodule_search_locations=[str(_package)])
_module = importlib.util.module_from_spec(_spec)
sys.modules[__name__] = _module
_spec.loader.exec_module(_module)
