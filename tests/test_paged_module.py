"""CPU: the compiled module of the paged operators is found by its exact name."""
import os
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
