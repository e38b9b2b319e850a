"""
Calls of the expert-layer operators at the edges of what they take: huge magnitudes, sizes next to a launch limit, several
host threads, row counts past a limit, waits that run out.  References and tolerances as in test_gpu_experts.py.
"""
import pytest

from ios.contrib import ios_runtime as rt

pytestmark = pytest.mark.gpu

torch = pytest.importorskip('torch')

from test_gpu_experts import BF16, F16, F32, U, generator, quantize_reference  # noqa: E402


# ---- quantiser: magnitudes whose products with 254 pass float32 ------------------------------------

def rows_of_halves(power, width, dtype):
    """All halves n + 1/2 below 127 of a row whose largest is 127, both signs, times a power of two: exact in every type."""
    halves = torch.arange(127, device='cuda').double() + 0.5
    row = torch.cat([halves, torch.tensor([127.0], dtype=torch.float64, device='cuda')]) * 2.0 ** power
    return torch.stack([row, -row]).repeat(1, width // 128).to(dtype)


@pytest.mark.parametrize('dtype', [BF16, F32], ids=['bf16', 'fp32'])
@pytest.mark.parametrize('power', [121, 120, 118, 93, 92, 0, -107, -108, -126])
@pytest.mark.parametrize('width', [128, 2048, 4096, 8192])
def test_quantized_halves_at_any_magnitude(dtype, power, width):
    x = rows_of_halves(power, width, dtype)
    q, scale = rt.quantize_rows(x)
    expect, expect_scale = quantize_reference(x)
    assert torch.equal(q.double(), expect)
    assert ((scale.double() - expect_scale).abs() <= U * expect_scale + 2.0 ** -150).all()
    odd = torch.cat([x, x], 1)[:, 1:width + 1]                  # element by element
    assert torch.equal(rt.quantize_rows(odd)[0].double(), quantize_reference(odd)[0])


@pytest.mark.parametrize('dtype', [F16, BF16, F32], ids=['fp16', 'bf16', 'fp32'])
def test_quantized_rows_of_huge_values(dtype):
    top = torch.finfo(dtype).max
    x = (torch.randn(200, 1000, generator=generator(21), device='cuda') * (top / 6)).clamp(-top, top).to(dtype)
    x[0, :3] = torch.tensor([top, top / 2, -top], device='cuda').to(dtype)
    x[1, 5], x[2, 6] = float('inf'), float('nan')
    for view in (x, x[:, 1:]):
        assert torch.equal(rt.quantize_rows(view)[0].double(), quantize_reference(view)[0])
