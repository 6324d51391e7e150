"""CPU checks of the build script, with a compiler that only makes its output file."""
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAKE = "#!/bin/sh\necho \"$0 $*\" >> \"$BUILD_LOG\"\nwhile [ $# -gt 0 ]; do [ \"$1\" = -o ] && : > \"$2\"; shift; done\n"


@pytest.fixture
def tree(tmp_path):
    """A copy of the package's build script and sources, with fakes of both compilers."""
    skip = shutil.ignore_patterns("_build", "__pycache__")
    shutil.copytree(os.path.join(ROOT, "moe_stream_b200"), tmp_path / "moe_stream_b200", ignore=skip)
    shutil.copytree(os.path.join(ROOT, "include"), tmp_path / "include")
    (tmp_path / "bin").mkdir()
    for name in ("nvcc", "g++"):
        (tmp_path / "bin" / name).write_text(FAKE)
        (tmp_path / "bin" / name).chmod(0o755)
    return tmp_path


def run(tree, path=()):
    """Runs the build; returns the names of the fakes' outputs and what was printed."""
    log = tree / "log"
    log.write_text("")
    env = dict(os.environ, NVCC=str(tree / "bin" / "nvcc"), BUILD_LOG=str(log), PATH=f"{tree / 'bin'}:{os.environ['PATH']}")
    env.pop("PYTHONPATH", None)
    code = f"import sys; sys.path[:0] = {[str(tree), *map(str, path)]!r}\n"
    if not path:
        code += "sys.modules['torch'] = None\n"                   # what is not installed
    p = subprocess.run([sys.executable, "-c", code + "from moe_stream_b200 import build; build.build()"], env=env, cwd=tree,
                       capture_output=True, text=True)
    assert p.returncode == 0, p.stderr
    made = [os.path.basename(line.split(" -o ")[1].split()[0]) for line in log.read_text().splitlines()]
    return made, p.stdout + p.stderr


def test_the_library_builds_without_torch(tree):
    made, said = run(tree)
    assert {"libmoestream_cuda.so", "libmoestream_cuda.a", "runtime.o"} <= set(made)
    assert "_binding.so" not in made and "torch is not installed" in said
    assert (tree / "moe_stream_b200" / "_build" / "libmoestream_cuda.a").exists()


def test_the_extension_is_built_again_for_another_torch(tree):
    at = tree / "site" / "torch"
    at.mkdir(parents=True)
    (at / "__init__.py").write_text("raise ImportError('the build imports no torch')")
    (at / "version.py").write_text("__version__ = '1'")
    assert "_binding.so" in run(tree, [tree / "site"])[0]
    assert run(tree, [tree / "site"])[0] == []                       # nothing is stale
    os.utime(at / "version.py", (0, 0))                              # older files, another version
    (at / "version.py").write_text("__version__ = '2'")
    os.utime(at / "version.py", (0, 0))
    assert run(tree, [tree / "site"])[0] == ["_binding.so"]


def test_an_extension_for_another_torch_is_not_loaded(monkeypatch, tmp_path):
    pytest.importorskip("torch")
    from moe_stream_b200 import _lib
    so, stamp = tmp_path / "_binding.so", tmp_path / "_binding.torch"
    monkeypatch.setattr(_lib, "BINDING_PATH", str(so))
    monkeypatch.setattr(_lib, "BINDING_TORCH", str(stamp))
    monkeypatch.setattr(_lib, "_binding", None)
    with pytest.raises(OSError, match="missing"):
        _lib.binding()
    so.write_text("")
    stamp.write_text("__version__ = '0'")
    with pytest.raises(OSError, match="another torch"):
        _lib.binding()
