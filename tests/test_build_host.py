"""What build.py asks of the machine: the C-ABI library needs nvcc alone, the Python binding
needs torch and g++ and is left out without them; builds at the same time do not write into
one another's files. Compilers are stand-ins that write what they were asked for."""
import importlib.util
import os
import subprocess
import sys
import threading

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def build(tmp_path, monkeypatch):
    spec = importlib.util.spec_from_file_location("gqa_build_copy", os.path.join(ROOT, "gqa-flash-attn-rtx3060_b200", "build.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    for name in ("OUT", "OUT_DEBUG", "EXT"):
        monkeypatch.setattr(mod, name, str(tmp_path / (name + ".so")))
    mod.commands = []
    real = subprocess.run

    def run(cmd, **kw):
        if os.path.basename(cmd[0]) not in ("nvcc", "g++"):
            return real(cmd, **kw)
        mod.commands.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write(os.path.basename(cmd[0]))
        return subprocess.CompletedProcess(cmd, 0)
    monkeypatch.setattr(mod.subprocess, "run", run)
    monkeypatch.setattr(mod, "nvcc", lambda: "/usr/local/cuda/bin/nvcc")
    return mod


def compilers(mod):
    return [os.path.basename(c[0]) for c in mod.commands]


def test_library_and_binding(build):
    assert build.build() == build.OUT and sorted(compilers(build)) == ["g++", "nvcc"]
    with open(build.EXT) as f:
        assert f.read().startswith("g++")
    build.commands.clear()
    assert build.build() == build.OUT and build.commands == []  # both up to date
    assert build.build(debug=True) == build.OUT_DEBUG and compilers(build) == ["nvcc"]


def test_the_library_builds_without_torch(build, monkeypatch):
    real = importlib.util.find_spec
    monkeypatch.setattr(build.importlib.util, "find_spec", lambda name, *a: None if name == "torch" else real(name, *a))
    assert build.build() == build.OUT and compilers(build) == ["nvcc"]
    assert os.path.exists(build.OUT) and not os.path.exists(build.EXT)


def test_the_library_builds_without_gxx(build, monkeypatch):
    real = build.shutil.which
    monkeypatch.setattr(build.shutil, "which", lambda name, *a: None if name == "g++" else real(name, *a))
    assert build.build() == build.OUT and compilers(build) == ["nvcc"] and not os.path.exists(build.EXT)


def test_the_binding_has_torchs_own_string_abi(build):
    import torch
    build.build()
    cmd = next(c for c in build.commands if os.path.basename(c[0]) == "g++")
    assert f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}" in cmd


def test_builds_at_the_same_time_write_their_own_files(build):
    threads = [threading.Thread(target=build.build, kwargs=dict(force=True, debug=d)) for d in (False, True)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    outs = [c[c.index("-o") + 1] for c in build.commands]
    assert len(outs) == len(set(outs)) == 4
    assert sorted(os.listdir(os.path.dirname(build.OUT))) == ["EXT.so", "OUT.so", "OUT_DEBUG.so"]


def test_the_real_build_is_importable_from_a_plain_interpreter():
    """build.py itself imports neither torch nor anything else that is not in the standard library."""
    code = f"import sys; sys.modules['torch'] = None; sys.path.insert(0, {os.path.join(ROOT, 'gqa-flash-attn-rtx3060_b200')!r}); import build"
    subprocess.run([sys.executable, "-c", code], check=True)
