"""Large matrices in the 4-bit microscaled formats, made on the GPU from their definition, with their values in fp64."""
import torch

BLOCK = {"mxfp4": 32, "nvfp4": 16}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def whole_matrix(rows, k, fmt, seed):
    """(matrix, fp64 values): whole numbers of at most 12 halves, times a power of two a row (nvfp4): sums of their products are exact in fp32."""
    from trellis_b200 import microscale
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(0, 16, (rows, k + k % 2), generator=g, device="cuda")
    up = torch.randint(0, 2, (rows, -(-k // BLOCK[fmt])), generator=g, device="cuda")
    row = None if fmt == "mxfp4" else torch.randint(-2, 3, (rows,), generator=g, device="cuda").float().exp2()
    q = microscale.from_blocks((codes[:, 0::2] | (codes[:, 1::2] << 4)).to(torch.uint8), (up + 127 if fmt == "mxfp4" else 0x38 + 8 * up).to(torch.uint8), row, k, fmt)
    v = torch.tensor(E2M1 + tuple(-e for e in E2M1), dtype=torch.float64, device="cuda")[codes[:, :k]]
    v *= (1.0 + up).double().repeat_interleave(BLOCK[fmt], 1)[:, :k]
    return q, v if row is None else v * row.double()[:, None]


def whole_tokens(m, k, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-8, 9, (m, k), generator=g, device="cuda").to(dtype)
