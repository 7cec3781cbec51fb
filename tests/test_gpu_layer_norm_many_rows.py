"""Layer norm of more rows than one launch holds threads for: 2^29 rows of 8 threads each are 2^32."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,W", [(torch.float32, 1), (torch.bfloat16, 2)])
def test_rows_past_the_threads_of_a_launch(dtype, W):
    from ocean import ops
    R = (1 << 29) + 37
    x = torch.empty(R, W, device="cuda", dtype=dtype)
    x[:] = torch.arange(1, W + 1, device="cuda", dtype=dtype)       # every row the same: xh is 0, or -1, 1 less eps's share
    w, b = torch.full((W,), 3.0, device="cuda"), torch.full((W,), 0.5, device="cuda")
    one = ops.layer_norm(x[:5], w, b)
    assert torch.equal(one[0].float(), torch.tensor([0.5] if W == 1 else [-2.5, 3.5], device="cuda"))
    assert (ops.layer_norm(x, w, b) == one[0]).all()
    y, s = ops.add_layer_norm(x, x, w, b)
    assert (s == 2 * x[0]).all() and (y == ops.add_layer_norm(x[:5], x[:5], w, b)[0][0]).all()
