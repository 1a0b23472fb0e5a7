"""When torch's side of the operators around the attention is built again: it is compiled against one torch."""
import os

import pytest

from dsalt_b200 import build


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """A library folder in which everything is newer than its sources; calls of the two builds are counted."""
    calls = []
    for name in ("OUT_DIR", "LIB", "TORCH_LIB"):
        at = os.path.basename(getattr(build, name))
        monkeypatch.setattr(build, name, str(tmp_path) if name == "OUT_DIR" else str(tmp_path / at))
    for path in (build.LIB, build.TORCH_LIB):
        open(path, "w").close()

    def torch_side(target):
        calls.append(target)
        open(target, "w").close()

    monkeypatch.setattr(build, "_build_kernels", lambda verbose: calls.append("kernels"))
    monkeypatch.setattr(build, "_run_compiler", torch_side)
    return calls


def test_torch_side_is_built_again_for_another_torch(tree, monkeypatch):
    import torch
    build.build()
    assert len(tree) == 1 and "kernels" not in tree  # of which torch it is was not noted
    build.build()
    assert len(tree) == 1
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    build.build()
    assert len(tree) == 2
    build.build()
    assert len(tree) == 2
    os.remove(build.TORCH_LIB)
    build.build()
    assert len(tree) == 3


def test_torch_side_takes_torchs_own_abi(monkeypatch):
    import torch
    for abi in (True, False):
        monkeypatch.setattr(torch._C, "_GLIBCXX_USE_CXX11_ABI", abi)
        assert f"-D_GLIBCXX_USE_CXX11_ABI={int(abi)}" in build._torch_command("out.so")
