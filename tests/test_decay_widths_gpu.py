"""decay_linear_attention at head dimensions that fill no tile, over chunks enough that loads are on their way for several of them at a time."""
import pytest

from test_decay_attention_gpu import _check, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dk,dv", [(80, 96), (128, 130), (40, 24), (3, 5), (200, 72), (8, 256)])
@pytest.mark.parametrize("B,T", [(2, 385), (1, 449)])
def test_many_chunks(B, T, dk, dv, dtype):
    """Seven and more chunks of 64."""
    _check(*_inputs(B, 2, T, dk, dv, dtype, token_first=True, seed=51))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dk,dv", [(80, 130), (20, 136)])
def test_many_chunks_of_a_segment(dk, dv, dtype):
    """24 walks of a row's segments: ten of 512 tokens, eight chunks of 64 and sixteen of 32."""
    _check(*_inputs(1, 8, 5000, dk, dv, dtype, decay=0.05, seed=52))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_many_chunks_of_packed_sequences(dtype):
    lens = [500, 0, 64, 321, 1, 448]
    _check(*_inputs(1, 2, sum(lens), 72, 40, dtype, rows=len(lens), seed=53), lens=lens)
