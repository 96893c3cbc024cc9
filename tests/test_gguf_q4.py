"""Q4_0 tensors of a GGUF file that are not whole: the file still reads, as it does for types that the
decode path does not know; only asking for their blocks fails."""
import numpy as np
import pytest

from test_gguf import _write_gguf


@pytest.mark.parametrize("shape,data", [((3, 11), b"\0" * 40), ((2, 64), b"\0" * 8)], ids=["not whole blocks", "cut short"])
def test_a_q4_0_tensor_that_is_not_whole(tmp_path, q3, shape, data):
    from q3b200 import gguf

    path = str(tmp_path / "a.gguf")
    good = np.arange(8, dtype=np.float32)
    _write_gguf(path, [("good", (8,), gguf.GGML_F32, good.tobytes()), ("odd", shape, gguf.GGML_Q4_0, data)])
    _, t = gguf.read_gguf(path)
    assert np.array_equal(np.array(t["good"][0]).view(np.float32), good)
    assert t["odd"][0] is None and t["odd"][1:] == (shape, gguf.GGML_Q4_0)
    with pytest.raises(gguf.GGUFError, match="odd"):
        gguf.q4_0(t, "odd", *shape)
