"""What the entry point of the log probabilities refuses before anything runs."""
import pytest

torch = pytest.importorskip("torch")

from relax_b200 import _lib


@pytest.mark.skipif(torch.cuda.is_available(), reason="the buffer is host memory")
@pytest.mark.parametrize("dtype", [_lib.F16, _lib.BF16, _lib.F32])
def test_rows_whose_indices_would_not_fit(dtype):
    """Near 2^31 entries a thread's index passes the largest whole number behind the row's end, and is less than the end again."""
    p = torch.zeros(64, dtype=torch.int32).data_ptr()
    call = _lib.lib().b200_token_logprobs
    for V in (2 ** 31 - 4096, 2 ** 31 - 300, 2 ** 31 - 66, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 5):
        for top in (0, 5):
            assert call(p, dtype, V, p, p, p, p, p, 1, V, top, None) == _lib.EINVAL, (V, top)
    assert call(p, dtype, 2 ** 31 - 4097, p, p, p, p, p, 1, 2 ** 31 - 4097, 5, None) == _lib.ENODEVICE
