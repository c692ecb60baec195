"""CPU: how the compiled module of the paged operators is built and found."""
import os
import subprocess
import sysconfig

import pytest


def test_only_this_pythons_module_is_loaded(tmp_path, monkeypatch):
    from polykernel_b200 import paged
    monkeypatch.setattr(paged, "_module", None)
    monkeypatch.setattr(paged, "LIB_PATH", str(tmp_path / "libpkb200.so"))
    (tmp_path / "_paged.cpython-37m-other.so").write_bytes(b"another version's")
    with pytest.raises(RuntimeError, match="not built"):
        paged.load_paged()
    here = "_paged" + sysconfig.get_config_var("EXT_SUFFIX")
    from polykernel_b200 import _lib
    for name in (here, "libpkb200.so"):
        os.symlink(os.path.join(os.path.dirname(_lib.LIB_PATH), name), tmp_path / name)
    assert hasattr(paged.load_paged(), "rope")


def test_the_library_builds_without_python(tmp_path):
    """`make` in csrc needs nvcc alone: its default target runs no Python."""
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "polykernel_b200", "csrc")
    plan = subprocess.run(["make", "-C", csrc, "-n", "-B"], capture_output=True, text=True, check=True).stdout
    assert "nvcc" in plan and "python" not in plan
    plan = subprocess.run(["make", "-C", csrc, "-n", "-B", "binding"], capture_output=True, text=True, check=True).stdout
    assert "build_binding" in plan


@pytest.mark.parametrize("name", ["rope", "rope_backward"])
def test_what_is_no_tensor_is_a_type_error(name):
    torch = pytest.importorskip("torch")
    from polykernel_b200 import ops
    call = getattr(ops, name)
    x, pos, f = torch.zeros(2, 1, 8), torch.zeros(2, dtype=torch.int64), torch.ones(4)
    for args in ((None, pos, f), (x, None, f), (x, pos, None)):
        with pytest.raises(TypeError):
            call(*args)
