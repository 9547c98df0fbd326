"""What the Python wrappers of the prompt operators refuse on device tensors."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16
FAR = 2 ** 32  # becomes 0 in the C entry points' 32-bit sizes, which is an empty call there


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def test_sizes_past_32_bits(qimg):
    """Expanded views have any size without memory; each would have returned an
    output that nothing was written to."""
    one = torch.zeros(1, 1, 64, dtype=BF, device=DEV)
    far = one.expand(FAR, 1, 64)
    with pytest.raises(qimg.QimgError, match="2\\^31"):
        qimg.attention_varlen(far, one, one, _i32(0, 1), _i32(0, 1), out=far)
    with pytest.raises(qimg.QimgError, match="2\\^31"):
        qimg.attention_varlen(one, far, far, _i32(0, 1), _i32(0, 1), out=one.clone())
    row = torch.zeros(1, 8, dtype=BF, device=DEV)
    col = torch.zeros(1, 1, dtype=BF, device=DEV)
    with pytest.raises(qimg.QimgError, match="2\\^31"):
        qimg.linear_forward_bf16_fused(row.expand(FAR, 8), row, out=col.expand(FAR, 1))
    table = torch.zeros(4, 4, 2, device=DEV)
    x = torch.zeros(1, 1, 8, device=DEV)
    with pytest.raises(qimg.QimgError, match="2\\^31"):
        qimg.rope_packed(x.expand(1, FAR, 8), table, _i32(0), 0, out=x.expand(1, FAR, 8))
    with pytest.raises(qimg.QimgError, match="2\\^31"):
        qimg.rope_packed(x, table, _i32(0), FAR + 1)
