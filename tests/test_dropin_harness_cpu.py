"""What the drop-in's tests do where their harness is missing: skip where onnx-light's sources are
missing too, fail where it could have been built."""
import pytest

import dropin


@pytest.fixture
def no_harness(monkeypatch, tmp_path):
    monkeypatch.setattr(dropin, "_lib", None)
    monkeypatch.setattr(dropin, "HARNESS", str(tmp_path / "libref_harness.so"))
    monkeypatch.setenv("ONNXL_REFERENCE", str(tmp_path))
    return tmp_path


def test_without_sources_it_skips(no_harness):
    with pytest.raises(pytest.skip.Exception, match="no onnx-light source tree"):
        dropin.lib()


def test_with_sources_it_fails(no_harness):
    (no_harness / "onnx_light").mkdir()
    with pytest.raises(FileNotFoundError, match="not built"):
        dropin.lib()
