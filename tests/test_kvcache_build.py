"""How the paged cache's native parts are built and loaded beside the rest."""
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "whisper-timestamped_amd")


def test_a_library_without_the_caches_entries_serves_the_others(tmp_path):
    """Entries may be added within an ABI version: a library that lacks the cache's is refused by the cache alone, one that lacks
    another is refused as a whole."""
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not found")
    from whisper_timestamped import _lib

    def built(name, entries):
        src, so = tmp_path / f"{name}.c", tmp_path / f"{name}.so"
        src.write_text("".join(f"int {e}(void) {{ return {_lib.ABI_VERSION if e == 'wt_version' else -3}; }}\n" for e in entries))
        subprocess.check_call([gcc, "-shared", "-fPIC", str(src), "-o", str(so)])
        return so

    def run(so, code):
        return subprocess.run([sys.executable, "-c", code], env=dict(os.environ, WT_LIBWTALIGN=str(so), PYTHONPATH=PKG), capture_output=True, text=True)

    others = [e for e in _lib.EXPORTS if not e.startswith("wt_kv_")]
    assert len(others) == len(_lib.EXPORTS) - 4
    p = run(built("older", others), "from whisper_timestamped import _lib, PagedKVCache\nL = _lib.load()\nassert L.wt_release_stream(None) == -3\n"
            "import torch\nk = torch.zeros(1, 1, 8, 64)\nPagedKVCache(k, k.clone())")
    assert p.returncode == 1 and "ImportError" in p.stderr and "wt_kv_append" in p.stderr, p.stderr
    p = run(built("broken", [e for e in _lib.EXPORTS if e != "wt_logmel_batch"]), "from whisper_timestamped import _lib\n_lib.load()")
    assert p.returncode == 1 and "ImportError" in p.stderr and "wt_logmel_batch" in p.stderr, p.stderr
