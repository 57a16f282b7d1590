"""attn_linear through the static scratch where two of its states do not fit it."""
import numpy as np
import pytest

from linear_cases import Linear
from test_gpu_linear import CHUNKS, TOKENS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("counts, chunks", [([33], True), ([223], True), ([224], False), ([200, 1, 130], False)])
def test_64_heads_of_128(gpu, counts, chunks):
    """Two states that passes would hand on are 8.06 MB. Seven chunks, of 1.1 MB each,
    fit the 8 MB of the scratch in one pass, with qmr_encode's bits (a launch counts
    tokens / 32 and one more for every sequence); more tokens go one after the
    other, and are right as well."""
    case = Linear(counts, 16, 64, 128, 128)
    out, after = case.check(gpu, CHUNKS)
    got, state = case.check(gpu, CHUNKS if chunks else TOKENS, static=True)
    assert gpu.last_hip_kernel() == ("linear_scan_kernel" if chunks else "attn_linear_tokens_kernel")
    if chunks:
        assert np.array_equal(got, out) and np.array_equal(state, after)
