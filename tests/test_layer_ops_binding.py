"""The compiled binding of an earlier build, which lacks operators that the library has, is not used.  CPU only."""
import importlib.util

import pytest
import torch

import moe_block as mb

NAMES = [n[len("moe_"):] for n, _ in mb._Entries._fields_]


@pytest.mark.parametrize("there, taken", [(NAMES, True), (NAMES[:6], False), (NAMES[:-1], False)])
def test_a_binding_without_every_operator_is_left(there, taken, tmp_path, monkeypatch):
    if getattr(torch._C, "_cuda_getCurrentRawStream", None) is None:
        pytest.skip("this torch has no raw streams: no binding is taken at all")
    path = tmp_path / "moe_torch.py"
    path.write_text("import torch\ntorch_version = torch.__version__.partition('+')[0]\n"
                    + "".join(f"def {n}(*a): return None\n" for n in ["set_current_stream", *there]))
    real = importlib.util.spec_from_file_location
    monkeypatch.setattr(mb.importlib.util, "spec_from_file_location", lambda name, _: real(name, path))
    monkeypatch.setattr(mb, "_row_types", {})
    monkeypatch.setattr(mb, "_torch_calls", None)
    mb._know_torch()
    assert (mb._torch_calls is not None) == taken
    assert mb._row_types[torch.bfloat16] == mb.GGML_BF16
