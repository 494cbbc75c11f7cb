"""The loaders of the compiled reference answer None, and build nothing, where there are no sources to build from."""
import pytest

import oracle_lib


@pytest.mark.parametrize("folder", [None, "empty", "src"])
@pytest.mark.parametrize("load", ["load_ref_host", "load_ref_cuda", "load_ref_matmul"])
def test_no_sources(load, folder, tmp_path, monkeypatch):
    root = tmp_path / "reference"
    if folder is not None:
        root.mkdir()
    if folder == "src":
        (root / "src").mkdir()
    monkeypatch.setattr(oracle_lib, "REFERENCE_ROOT", root)
    monkeypatch.setattr(oracle_lib, "ORACLE_DIR", tmp_path)
    monkeypatch.setattr(oracle_lib, "_make", lambda target: pytest.fail(f"make {target} without sources"))
    assert getattr(oracle_lib, load)() is None
