"""Shared pieces of the tests of 4-bit microscaled (MX4) matrices: the definition in 64 bits and the documented layout."""
import torch

LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def blocks_of(v):
    """Rows in blocks of 32, the last filled up with zeros."""
    return torch.nn.functional.pad(v.double(), (0, -v.shape[1] % 32)).reshape(v.shape[0], -1, 32)


def rounded(v):
    """Codes (rows x blocks x 32) and scale bytes (rows x blocks) of v's rows, from the definition: the nearest level of
    all eight by its distance, of two the one with an even index."""
    b = blocks_of(v)
    top = b.abs().amax(2)
    bad = ~torch.isfinite(top)
    mantissa, exponent = torch.frexp(torch.where(bad | (top == 0), torch.ones_like(top), top))
    e = torch.clamp(torch.where(top == 0, torch.full_like(exponent, -127), exponent - 1 - 2), min=-127)
    y = torch.where(bad[:, :, None], torch.zeros_like(b), b) * torch.exp2(-e.double())[:, :, None]
    levels = LEVELS.to(v.device)
    distance = (y.abs()[..., None] - levels).abs()
    # (an odd index loses a tie: no other difference of two distances is as small as this)
    distance = distance + torch.arange(8, device=v.device) % 2 * 1e-40
    least = distance.amin(-1, keepdim=True)
    tied = (distance == least).double() * (2.0 - torch.arange(8, device=v.device) % 2)
    code = tied.argmax(-1) + 8 * torch.signbit(b)
    code = torch.where(bad[:, :, None], torch.zeros_like(code), code)
    return code, torch.where(bad, torch.full_like(e, 255), e + 127)


def values(code, scale, cols):
    """What codes and scale bytes stand for, rows x cols."""
    levels = LEVELS.to(code.device)
    v = torch.where(code >= 8, -levels[code % 8], levels[code % 8])
    unit = torch.where(scale == 255, torch.full(scale.shape, float("nan"), dtype=torch.float64, device=code.device),
                       torch.exp2(scale.double() - 127))
    return (v * unit[:, :, None]).reshape(code.shape[0], -1)[:, :cols]


def buffer_of(code, scale, cols):
    """The MX4 matrix's bytes, placed one by one as the header says."""
    rows, device = code.shape[0], code.device
    chunks = (cols + 255) // 256
    out = torch.zeros((rows + 15) // 16 * chunks * 2176, dtype=torch.uint8, device=device)
    r = torch.arange(rows, device=device)[:, None]
    c = torch.arange(0, code.shape[1] * 32, 2, device=device)[None, :]
    unit = ((r // 16) * chunks + c // 256) * 2176
    lane = r % 16 + 16 * (c % 128 // 32)
    pairs = code.reshape(rows, -1)
    out[unit + 1024 * (c % 256 // 128) + 16 * lane + c % 32 // 2] = (pairs[:, ::2] | pairs[:, 1::2] << 4).to(torch.uint8)
    c = torch.arange(0, code.shape[1] * 32, 32, device=device)[None, :]
    unit = ((r // 16) * chunks + c // 256) * 2176
    lane = r % 16 + 16 * (c % 128 // 32)
    out[unit + 2048 + 2 * lane + c % 256 // 128] = scale.to(torch.uint8)
    return out


def matrix(v):
    """(the MX4 matrix's bytes, the values that it holds) of v's rows."""
    code, scale = rounded(v)
    return buffer_of(code, scale, v.shape[1]), values(code, scale, v.shape[1])


def exact_matrix(seed, rows, cols):
    """An MX4 matrix whose products' sums over at most 4096 columns are exact in 32 bits: multiples of 1/4 below 2^4."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    blocks = (cols + 31) // 32
    code = torch.randint(0, 16, (rows, blocks * 32), generator=g, device="cuda")
    code[:, cols:] = 0
    code = code.reshape(rows, blocks, 32)
    scale = torch.randint(126, 129, (rows, blocks), generator=g, device="cuda")
    return buffer_of(code, scale, cols), values(code, scale, cols)
