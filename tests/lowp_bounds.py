"""What the sums of linear_q4 may be off by, and inputs on which they have to be exact (used by the GPU tests, and by the CPU tests that show what they reject)."""
import torch

U = 2.0 ** -24                                             # fp32: half a step


def split(codes):
    return torch.stack([codes & 15, codes >> 4], -1).view(codes.shape[0], -1).double()


def q4_sums(x, codes, scales, zeros, group, waves=8):
    """(product in 64 bits, bound of its error) for sums that are kept in fp32, first over a group, then over the groups.

    Group g: the products x q are exact (16 bits by 4), each of its `group` additions - and each of those of sum x - is off by at most a step, 2 U, of a
    partial sum no larger than the sum of magnitudes; taking the zero point out rounds once more.  The groups' contributions s (sum q x - z sum x) are added
    by fused multiply-adds in `waves` chains, which are then added up: half a step each, of a partial sum no larger than the contributions' magnitudes."""
    N, G = scales.shape
    M = x.shape[0]
    q, s = split(codes).view(N, G, group), scales.double()
    z = torch.full_like(s, 8.0) if zeros is None else zeros.double()
    xg = x.double().view(M, G, group)
    y, err, mag = (torch.zeros(M, N, dtype=torch.float64) for _ in range(3))
    for g in range(G):
        a = xg[:, g] @ q[:, g].t().contiguous() - xg[:, g].sum(1, keepdim=True) * z[:, g]
        b = xg[:, g].abs() @ q[:, g].t().contiguous() + xg[:, g].abs().sum(1, keepdim=True) * z[:, g]
        y += a * s[:, g]
        err += (2 * group + 4) * U * b * s[:, g].abs()
        mag += (a * s[:, g]).abs()
    return y, err + (G + waves + 2) * U * (mag + err)


def whole_numbers(g, M, N, K, group, zeros, dtype):
    """(x, codes, scales, zeros) whose every partial sum is a multiple of 1 / 8 below 2^21: fp32 sums are exact in any order (K <= 11008:
    11008 x 8 x 15 / 2^-3 < 2^24)."""
    assert K <= 11008
    x = (torch.randint(1, 9, (M, K), generator=g) * (2 * torch.randint(0, 2, (M, K), generator=g) - 1)).to(dtype)      # (no zeros: every column counts)
    codes = torch.randint(0, 256, (N, K // 2), generator=g).to(torch.uint8)
    scales = torch.exp2(-torch.randint(0, 4, (N, K // group), generator=g).float()).to(dtype)
    return x, codes, scales, torch.randint(0, 16, (N, K // group), generator=g).to(torch.uint8) if zeros else None
