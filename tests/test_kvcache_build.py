"""How the paged cache's native parts are built and loaded beside the rest."""
import glob
import os
import re
import shutil
import subprocess
import sys
import sysconfig

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "whisper-timestamped_amd")
CSRC = os.path.join(PKG, "csrc")


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


def dry(*args):
    p = subprocess.run(["make", "-n", "-B", "-C", CSRC, *args], capture_output=True, text=True)
    assert p.returncode == 0, p.stderr
    return p.stdout


@pytest.mark.skipif(shutil.which("make") is None, reason="make not found")
def test_the_library_needs_no_torch():
    for out in (dry("lib"), dry("PY=false")):                # a Python without torch, or none
        assert "libwtalign.so" in out and "wt_kv_calls.cpp" not in re.sub(r"(?m)^echo.*$", "", out)
    assert "wt_kv_calls.cpp" in dry()


def test_the_calls_are_built_for_this_interpreter():
    """Named for the interpreter, so that another Python does not load them, and no untagged build beside them that it would."""
    found = [os.path.basename(f) for f in glob.glob(os.path.join(PKG, "whisper_timestamped", "_kvcalls*.so"))]
    assert found == ["_kvcalls" + sysconfig.get_config_var("EXT_SUFFIX")]


@pytest.mark.skipif(shutil.which("make") is None, reason="make not found")
def test_the_calls_are_rebuilt_for_another_torch(tmp_path):
    """What they were built for is kept in a file; they are out of date when it says something else."""
    csrc = tmp_path / "w" / "csrc"
    shutil.copytree(CSRC, csrc, ignore=shutil.ignore_patterns("*.o"))
    shutil.copytree(os.path.join(ROOT, "include"), tmp_path / "include")
    os.mkdir(tmp_path / "w" / "whisper_timestamped")

    def calls(*args):
        p = subprocess.run(["make", "-C", str(csrc), "calls", "CXX=true", *args], capture_output=True, text=True)
        assert p.returncode == 0, p.stderr
        for line in p.stdout.splitlines():                    # (the compiler does nothing here: its output file is made by hand)
            m = re.search(r"-o (\S*_kvcalls\S*\.so)", line)
            if m:
                (csrc / m.group(1)).resolve().touch()
        return "wt_kv_calls.cpp" in p.stdout

    assert calls() and not calls()
    assert calls("BUILT_FOR=another") and not calls("BUILT_FOR=another")
    assert calls()
