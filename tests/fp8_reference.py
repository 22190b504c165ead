"""What the tests of the 8-bit block operators compare with: the definition, written out in torch on the CPU, products in
64 bits."""
import torch

TOP = {"fp8_e4m3": 448.0, "fp8_e5m2": 57344.0}
DT = {"fp8_e4m3": torch.float8_e4m3fn, "fp8_e5m2": torch.float8_e5m2}


def quantize(x, fmt, tile=False):
    """(codes as float64 values, scales [K blocks, rows or row blocks] fp32, value of each element in float64)"""
    x = x.detach().cpu().float()
    rows, k = x.shape
    step = 128 if tile else 1
    codes = torch.empty(rows, k)
    scales = torch.empty(-(-k // 128), -(-rows // step))
    value = torch.empty(rows, k, dtype=torch.float64)
    for kb in range(scales.shape[0]):
        for rb in range(scales.shape[1]):
            block = x[rb * step:(rb + 1) * step, kb * 128:(kb + 1) * 128]
            s = torch.maximum(block.abs().max(), torch.tensor(2.0 ** -100)) * torch.tensor(1.0 / TOP[fmt], dtype=torch.float32)
            q = (block * (torch.ones(()) / s)).clamp(-TOP[fmt], TOP[fmt]).to(DT[fmt]).float()
            codes[rb * step:(rb + 1) * step, kb * 128:(kb + 1) * 128] = q
            scales[kb, rb] = s
            value[rb * step:(rb + 1) * step, kb * 128:(kb + 1) * 128] = q.double() * s.double()
    return codes.double(), scales, value


def product_bound(a, b, dtype, bias=None):
    """(a b^T + bias, how far a result in `dtype` may be from it) for values a [M, K], b [N, K] in float64.

    A sum over 128 products is formed by the tensor core to within 2^-22 of the sum of magnitudes (as its block-scaled form
    is); scaling it and adding it to the running sum in fp32 rounds three times per K block (the product of the scales, its product
    with the block's sum fused with the addition, and the addition where CTAs join), each at most 2^-24 of the sum of
    magnitudes so far; the bias adds one more, and the result is rounded once to its type."""
    y, mag = a @ b.t(), a.abs() @ b.abs().t()
    if bias is not None:
        y, mag = y + bias.double(), mag + bias.double().abs()
    blocks = -(-a.shape[1] // 128)
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    fp32 = (2.0 ** -22 + (3 * blocks + 2) * 2.0 ** -24) * mag
    return y, fp32 + (y.abs() + fp32) * torch.finfo(dtype).eps / 2 + tiny
