"""`import ah_rag` with the repository's root on the path: the package lies in ah-rag_amd/ah_rag, whose folder's
name a program would otherwise have to put on its path first. The import gives that package itself."""
import importlib.util
import os
import sys

_at = os.path.join(os.path.dirname(os.path.abspath(__file__)), "ah-rag_amd", "ah_rag")
_spec = importlib.util.spec_from_file_location(__name__, os.path.join(_at, "__init__.py"), submodule_search_locations=[_at])
_package = importlib.util.module_from_spec(_spec)
sys.modules[__name__] = _package  # (the import system hands out what stands here when this file ends)
try:
    _spec.loader.exec_module(_package)
except BaseException:
    sys.modules.pop(__name__, None)
    raise
