"""4-bit matrices and weights put together by a caller: kernels read as many bytes as the sizes say, on the GPU."""

import pytest
import torch

from flex_shard_amd.mxfp4 import MxFp4Matrix, MxFp4Weight, mxfp4_linear, mxfp4_quantize, quantize_mxfp4_weight


def test_a_matrix_has_its_bytes():
    whole = torch.zeros(3 * 2 * 136, dtype=torch.uint8)
    matrix = MxFp4Matrix(whole, 3, 300)
    assert matrix.data.shape == (3, 256) and matrix.scales.shape == (2, 3, 8)
    MxFp4Matrix(whole[:0], 0, 300)
    MxFp4Matrix(whole[:0], 3, 0)
    for buffer, rows, cols in (
        (whole[:-1], 3, 300), (whole, 4, 300), (whole, 3, 513), (whole, 3, 256), (whole.view(torch.int8), 3, 300), (whole.float(), 3, 300),
        (whole.view(3, -1), 3, 300), (torch.zeros(2 * 3 * 2 * 136, dtype=torch.uint8)[::2], 3, 300), (whole, -3, -300),
    ):
        with pytest.raises(ValueError, match="uint8"):
            MxFp4Matrix(buffer, rows, cols)


def test_a_weight_has_its_shape():
    def matrix(rows, cols):
        return MxFp4Matrix(torch.zeros(rows * -(-cols // 256) * 136, dtype=torch.uint8), rows, cols)

    MxFp4Weight((40, 64), torch.float32, matrix(40, 64), matrix(64, 40))
    MxFp4Weight((8, 40, 64), torch.float32, matrix(320, 64), matrix(512, 40))
    for shape, form, transposed in (
        ((40, 65), matrix(40, 64), None), ((41, 64), matrix(40, 64), None), ((8, 40, 64), matrix(40, 64), None), ((64,), matrix(1, 64), None),
        ((40, 64), matrix(40, 64), matrix(40, 64)), ((8, 40, 64), matrix(320, 64), matrix(64, 320)),
    ):
        with pytest.raises(ValueError, match="weight"):
            MxFp4Weight(shape, torch.float32, form, transposed)


def test_nothing_is_read_off_the_gpu():
    with pytest.raises(RuntimeError, match="no CPU path"):
        MxFp4Matrix(torch.zeros(136, dtype=torch.uint8), 1, 256).dequantize()


@pytest.mark.gpu
def test_from_bytes_and_back(device):
    w = torch.randn(40, 300, device=device)
    frozen = quantize_mxfp4_weight(w)
    kept = frozen.matrix.buffer.cpu()  # as a file would hold it
    again = MxFp4Weight((40, 300), w.dtype, MxFp4Matrix(kept.to(device), 40, 300))
    x = torch.randn(5, 300, device=device)
    with torch.no_grad():
        assert torch.equal(mxfp4_linear(x, again), mxfp4_linear(x, frozen))
    assert torch.equal(again.matrix.dequantize(torch.float32), mxfp4_quantize(w).dequantize(torch.float32))
    with pytest.raises(RuntimeError, match="no CPU path"):
        MxFp4Matrix(kept, 40, 300).dequantize()
