"""`import q4rdna` for programs started in the repository's root.

The package lives in rdna-gfx1201-v0.1_amd/, a folder whose name is no package
name; this module puts the package in its own place.  Programs that have that
folder on their path get the package directly.
"""
import importlib.util
import os
import sys

_PACKAGE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "rdna-gfx1201-v0.1_amd", "q4rdna")
_spec = importlib.util.spec_from_file_location("q4rdna", os.path.join(_PACKAGE, "__init__.py"),
                                               submodule_search_locations=[_PACKAGE])
_module = importlib.util.module_from_spec(_spec)
sys.modules["q4rdna"] = _module
_spec.loader.exec_module(_module)
