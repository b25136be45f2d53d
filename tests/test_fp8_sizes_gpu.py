"""8-bit blocks of matrices with as many columns as an int counts."""
import pytest
import torch

import fp8_oracle as fo
from test_fp8_gpu import L, call  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("K", [2 ** 31 - 16, 2 ** 31 - 256])
def test_a_matrix_of_one_long_row(kge, L, K):
    g = torch.Generator().manual_seed(7)
    w = torch.zeros(K, dtype=torch.bfloat16, device="cuda")
    tail = torch.randn(1024 + K % 128, generator=g).to(torch.bfloat16)      # whole blocks from its beginning on
    begin = K - len(tail)
    assert begin % 128 == 0
    w[begin:] = tail.cuda()
    blocks = -(-K // 128)
    codes, scales = torch.full((K + 16,), 0x55, dtype=torch.uint8, device="cuda"), torch.full((blocks + 1,), 9.0, device="cuda")
    call(kge, "kge_fp8_quant_weight", codes, scales, w, 1, 1, K)
    torch.cuda.synchronize()
    code, scale = fo.quantise(tail[None], 1)
    assert torch.equal(codes[begin:K].cpu().view(fo.E4M3).double(), code[0]) and torch.equal(scales[begin // 128:blocks].cpu(), scale[0].float())
    assert not codes[:begin].any() and (scales[:begin // 128] == fo.LEAST).all() and (codes[K:] == 0x55).all() and scales[blocks] == 9
