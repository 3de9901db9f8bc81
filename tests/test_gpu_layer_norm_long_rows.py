"""Layer norm of rows too long for registers, many of them: their column sums run over up to 64 rows a thread.
Bars as in test_gpu_layer_norm."""

import pytest
import torch

from test_gpu_layer_norm import check_backward, check_forward, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,width,dtype,w_dtype", [(4096, 16392, torch.bfloat16, torch.bfloat16),
                                                      (3001, 16385, torch.bfloat16, torch.float32),
                                                      (700, 33333, torch.float16, torch.float16),
                                                      (513, 20001, torch.float32, torch.float32)])
def test_many_long_rows(rows, width, dtype, w_dtype):
    x, w, b, dy = inputs(rows, width, dtype, w_dtype)
    check_forward(x, w, b)
    check_backward(dy, x, w, b)
