"""The 4-bit microscaled formats from their definition, in 64 bits with torch on the CPU: what the kernels are tested against."""
import math

import torch

BLOCK = {"mxfp4": 32, "nvfp4": 16}
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
BORDERS = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)


def nearest_e2m1(q):
    """Codes (sign in bit 3) of the nearest values: ties to the even code, beyond 6 to 6."""
    a, code = q.abs(), torch.zeros(q.shape, dtype=torch.int64)
    for i, border in enumerate(BORDERS):
        code += (a > border) if i % 2 == 0 else (a >= border)       # the code below border i is i: a tie goes up from an odd one
    return code + 8 * torch.signbit(q)


def nearest_e4m3(t):
    """Bytes of the nearest e4m3 numbers of 0 <= t <= 448 (ties to even), and their values."""
    _, e = torch.frexp(t)
    e = (e - 1).clamp(min=-6)
    m = torch.round(torch.ldexp(t, 3 - e))                          # eighths: 0 .. 16 (torch.round: ties to even)
    v = torch.ldexp(m, e - 3)
    up = m == 16
    e, m = torch.where(up, e + 1, e), torch.where(up, 8.0, m)
    return torch.where(m < 8, m, (e + 7) * 8 + m - 8).to(torch.int64), v


def quantize(x, fmt):
    """(codes int64 [rows, k], scale bytes int64 [rows, blocks], row scales fp64 [rows] or None) of a CPU matrix."""
    rows, k = x.shape
    b = BLOCK[fmt]
    v = torch.nn.functional.pad(x.double(), (0, -k % b)).reshape(rows, -1, b)
    fine = torch.isfinite(v)
    good = fine.all(2)
    amax = torch.where(good[..., None], v, torch.zeros_like(v)).abs().amax(2)
    row = None
    if fmt == "mxfp4":
        e = (torch.frexp(amax)[1] - 1 - 2).clamp(min=-127)
        e = torch.where(amax > 0, e, -127)
        byte, d = e + 127, torch.ldexp(torch.ones_like(amax), e)
        nan = 255
    else:
        top = torch.where(fine, v, torch.zeros_like(v)).abs().amax(2).amax(1)
        j = torch.full((rows,), -80, dtype=torch.int64)
        while bool((over := top > torch.ldexp(torch.full_like(top, 2688.0), j)).any()):
            j += over
        j = torch.where(top > 0, j, 0)
        row = torch.ldexp(torch.ones(rows, dtype=torch.float64), j)
        byte, s = nearest_e4m3(amax / row[:, None] / 6)
        d = s * row[:, None]
        nan = 0x7F
    q = torch.where(d[..., None] > 0, v / d[..., None].clamp(min=1e-300), v * 0.0)
    codes = nearest_e2m1(torch.where(good[..., None], q, torch.zeros_like(q)))
    return codes.reshape(rows, -1)[:, :k], torch.where(good, byte, nan), row


def scale_values(byte, fmt):
    if fmt == "mxfp4":
        return torch.where(byte == 255, math.nan, torch.ldexp(torch.ones(byte.shape, dtype=torch.float64), byte - 127))
    e, m = byte >> 3, (byte & 7).double()
    v = torch.where(e == 0, torch.ldexp(m, torch.full_like(e, -9)), torch.ldexp(8 + m, e - 10))
    return torch.where(byte == 0x7F, math.nan, v)


def values(codes, byte, row, fmt):
    """fp64 [rows, k]."""
    v = torch.tensor(VALUES, dtype=torch.float64)[codes & 7] * torch.where(codes >= 8, -1.0, 1.0)
    v = v * scale_values(byte, fmt).repeat_interleave(BLOCK[fmt], 1)[:, :codes.shape[1]]
    return v if row is None else v * row.double()[:, None]


def unpack(q):
    """(codes, scale bytes, row scales) of a ``Microscaled`` matrix, read byte by byte from its storage as documented."""
    rows, k = q.shape
    c = q.codes.cpu().to(torch.int64)
    codes = torch.stack((c & 15, c >> 4), 2).reshape(rows, -1)
    assert not codes[:, k:].any(), "codes behind the last column"
    nb = -(-k // BLOCK[q.fmt])
    s = q.scales.cpu().to(torch.int64)
    r, b = torch.arange(rows)[:, None], torch.arange(s.shape[1] * 4)[None, :]
    byte = s[r // 128, b // 4, r % 32, r % 128 // 32, b % 4]
    assert not byte[:, nb:].any(), "scales behind the last column"
    return codes[:, :k], byte[:, :nb], None if q.row_scale is None else q.row_scale.cpu().double()


def pack(codes, byte, row, fmt, device="cpu"):
    """A ``Microscaled`` matrix of given codes and scales, written as documented; scales of rows that do not exist are NaN."""
    from trellis_b200 import microscale
    rows, k = codes.shape
    c = torch.zeros(rows, 32 * -(-k // 32), dtype=torch.int64)
    c[:, :k] = codes
    c = (c[:, 0::2] | (c[:, 1::2] << 4)).to(torch.uint8)
    atoms = (4 if fmt == "nvfp4" else 2) * -(-k // 256)
    s = torch.zeros(-(-rows // 128), atoms, 32, 4, 4, dtype=torch.uint8)
    full = torch.full((s.shape[0] * 128, atoms * 4), 255 if fmt == "mxfp4" else 0x7F, dtype=torch.uint8)
    full[:rows] = 0
    full[:rows, :byte.shape[1]] = byte.to(torch.uint8)
    r, b = torch.arange(s.shape[0] * 128)[:, None], torch.arange(atoms * 4)[None, :]
    s[r // 128, b // 4, r % 32, r % 128 // 32, b % 4] = full
    row = None if row is None else row.float().to(device)
    return microscale.Microscaled(c.to(device), s.to(device), row, (rows, k), fmt)


def random_matrix(rows, k, fmt, gen, spread=3):
    """Codes uniform, scales within 2^+-spread of 1, row scales powers of two."""
    codes = torch.randint(0, 16, (rows, k), generator=gen)
    nb = -(-k // BLOCK[fmt])
    if fmt == "mxfp4":
        return codes, torch.randint(127 - spread, 128 + spread, (rows, nb), generator=gen), None
    byte = torch.randint((7 - spread) * 8, (8 + spread) * 8, (rows, nb), generator=gen)
    return codes, byte, torch.ldexp(torch.ones(rows), torch.randint(-3, 4, (rows,), generator=gen))


def hadamard_blocks(x, signs, b):
    """Signs, then the orthonormal Sylvester-Hadamard transform of every b columns (fp64)."""
    h = torch.ones(1, 1, dtype=torch.float64)
    while h.shape[0] < b:
        h = torch.cat((torch.cat((h, h), 1), torch.cat((h, -h), 1)), 0)
    v = x.double() * signs.double()
    return (v.reshape(x.shape[0], -1, b) @ h / math.sqrt(b)).reshape(x.shape)
