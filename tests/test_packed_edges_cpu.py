"""Edges of the packed-sequence operators and of the encoder on them that need no GPU."""
import os
import subprocess
import sys

import pytest


@pytest.mark.parametrize("path", [["."], ["ah-rag_amd"], [".", "ah-rag_amd"], ["ah-rag_amd", "."]], ids="+".join)
def test_the_package_imports_from_the_repository_root(path):
    """With the root, the package's folder or both on the path, in either order: the same package, once."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    prog = ("import sys; sys.path[:0] = %r\n"
            "import ah_rag, ah_rag.packed, importlib\n"
            "from ah_rag.packed import packed_attention\n"
            "assert sys.modules['ah_rag'] is ah_rag and ah_rag.packed is sys.modules['ah_rag.packed']\n"
            "assert packed_attention is ah_rag.packed.packed_attention and importlib.import_module('ah_rag') is ah_rag\n"
            "print(ah_rag.__file__, ah_rag.packed.__file__, list(ah_rag.__path__))" % [os.path.join(root, p) for p in path])
    # (-I: neither the working folder nor PYTHONPATH)
    out = subprocess.run([sys.executable, "-I", "-c", prog], capture_output=True, text=True, timeout=300, cwd="/")
    assert out.returncode == 0, out.stderr
    init, packed, _ = (os.path.normpath(x) for x in out.stdout.split()[:3])
    pkg = os.path.join(root, "ah-rag_amd", "ah_rag")
    assert init == os.path.join(pkg, "__init__.py") and packed == os.path.join(pkg, "packed.py")
