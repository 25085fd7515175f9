"""Inputs of 4-bit linears whose every fp32 sum is exact, so that results are compared for equality
(test infrastructure).

Activations are small whole numbers, of one sign in a row, with at least one in every 32 inputs;
scales are powers of two from 2^-2; so each product and sum is a multiple of 2^-2, and exact while it
stays under 2^22 (`Linear.largest`).  Few activations are not zero, so that results are small
and a wrong term is not lost in the one rounding of the result."""
import torch

TERMS = 512  # activations of a row that are not zero, where each 32 inputs need no more than that
LONG_GROUPS = [(2_097_216, 2_097_184), (7_680_256, 1_280_032), (8_388_608, 4_194_336)]  # (K, group)
# more groups than LDS holds at a time: K in more ranges, or scales staged in rounds (many rows, or
# more groups in each of the ranges)
MANY_GROUPS = [(400, 5000, 12224, 96), (4000, 500, 4224, 32), (2100, 1024, 13824, 32), (33, 30000, 8224, 64),
               (3001, 2999, 8224, 64), (3000, 3000, 12224, 96), (3000, 3000, 20000, 128), (9000, 1000, 4224, 32), (100, 70, 70016, 32)]
# (m, n, k, group): every kernel and both their dtypes' forms: rows at and past the 16-row tiles, N that
# ends inside a tile, K of one block, inside a step of 128 inputs, in staged chunks and in ranges,
# groups of every alignment, a last group that is shorter
SHAPES = [(1, 1, 32, 32), (1, 16, 128, 128), (1, 1000, 5120, 128), (2, 33, 160, 64), (3, 77, 416, 96), (15, 50, 4096, 32),
          (16, 129, 1088, 128), (17, 64, 2080, 64), (31, 100, 96, 256), (32, 17, 992, 32), (33, 48, 1312, 160),
          (48, 250, 640, 128), (64, 31, 2016, 64), (65, 100, 512, 512), (130, 40, 288, 64), (1, 5000, 2048, 64),
          (1, 40, 16416, 32), (3, 40, 16416, 32), (4, 9000, 4256, 128), (2, 9000, 1056, 32), (20, 40, 16416, 32),
          (1, 20, 36864, 128), (2, 20, 36896, 256), (9, 9000, 544, 64), (40, 9000, 1056, 96),
          (17, 200, 1696, 64), (24, 512, 5120, 128), (33, 100, 8224, 32), (64, 300, 14336, 128), (100, 70, 70016, 32),
          (45, 20000, 544, 128), (200, 65, 1120, 96), (1, 13824, 5120, 64), (24, 5120, 13824, 128), (12, 1024, 5120, 32),
          (32, 13824, 5120, 128), (16, 2100, 70016, 64), (1, 9000, 32992, 32)]
BASE = {torch.bfloat16: 128, torch.float16: 1024}  # a code q is multiplied as BASE + q


class Linear:
    def __init__(self, m, n, k, group, dtype, zeros, bias, seed=0):
        g = torch.Generator().manual_seed(seed + m * 7 + n + k)
        self.m, self.n, self.k, self.group, self.dtype = m, n, k, group, dtype
        blocks, groups = k // 32, -(-k // group)
        if blocks > 8192:  # only some: the first and last of each group among them
            per = group // 32
            ends = torch.arange(groups) * per
            some = torch.cat((ends, ends + per - 1, torch.tensor([blocks - 1]), torch.randint(blocks, (200,), generator=g)))
            some = some[some < blocks].unique()
        else:
            some = torch.arange(blocks)
        count = min(32, max(1, TERMS // blocks))
        places = torch.rand(len(some), 32, generator=g).argsort(1)[:, :count]
        cols = (some[:, None] * 32 + places).flatten().sort().values  # inputs that some row has
        self.cols = cols
        self.x_cols = torch.randint(1, 4, (m, len(cols)), generator=g).double() * torch.where(torch.rand(m, 1, generator=g) < 0.5, -1, 1)
        self.codes = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
        self.scales = torch.tensor([0.25, 0.5, 1.0, 2.0])[torch.randint(0, 4, (n, groups), generator=g)].to(dtype)
        self.zeros = torch.randint(0, 16, (n, groups), generator=g, dtype=torch.uint8) if zeros else None
        self.bias = torch.randint(-50, 50, (n,), generator=g).to(dtype) if bias else None

    @property
    def x(self):
        x = torch.zeros(self.m, self.k, dtype=self.dtype)
        x[:, self.cols] = self.x_cols.to(self.dtype)
        return x

    def weight_cols(self, at=None):
        """(q - z) s of the inputs that are not zero, from the definition, in 64 bits; at: their groups."""
        q = self.codes[:, self.cols // 2].int()
        q = torch.where(self.cols % 2 == 0, q % 16, q // 16).double()
        at = self.cols // self.group if at is None else at
        z = 8.0 if self.zeros is None else self.zeros[:, at].double()
        return (q - z) * self.scales[:, at].double()

    def want(self, weight=None):
        y = self.x_cols @ (self.weight_cols() if weight is None else weight).t()
        return (y if self.bias is None else y + self.bias.double()).to(self.dtype)

    def largest(self):
        """What no product or sum passes: a row's terms and, under them, one step of 128 inputs with
        its codes as BASE + q (at most 39 + BASE for the difference and the zero point's part)."""
        terms = self.x_cols.abs() @ self.weight_cols().abs().t()
        step = torch.zeros(self.m, -(-self.k // 128), dtype=torch.float64).index_add_(1, self.cols // 128, self.x_cols.abs())
        return float(terms.max() + step.max() * 2 * (BASE[self.dtype] + 39)) + 50


def dense(m, n, k, group, dtype, seed=0, device="cpu"):
    """Ordinary inputs (x, codes, scales, zeros), and y in 64 bits.  A result of fp32 sums differs from y
    by less than one unit of dtype's rounding in norm: rounding many numbers takes 0.4 of one (it is
    the largest relative error of one number), and sums of about +-BASE sqrt(128) a group that err by
    2^-24 each some 2^-24 2 BASE / 4.6 of y, a twentieth of a unit, at any K."""
    g = torch.Generator(device=device).manual_seed(seed + m + n + k)
    groups = -(-k // group)
    codes = torch.randint(0, 256, (n, k // 2), generator=g, device=device, dtype=torch.uint8)
    scales = (torch.rand(n, groups, generator=g, device=device) * 0.02 + 1e-3).to(dtype)
    zeros = torch.randint(0, 16, (n, groups), generator=g, device=device, dtype=torch.uint8)
    x = torch.randn(m, k, generator=g, device=device).to(dtype)
    y = torch.zeros(m, n, dtype=torch.float64, device=device)
    for first in range(0, k, 4096 // group * group or group):  # whole groups at a time
        at = torch.arange(first, min(k, first + (4096 // group * group or group)), device=device)
        q = torch.stack((codes[:, at[::2] // 2] % 16, codes[:, at[::2] // 2] // 16), 2).flatten(1).double()
        y += x[:, at].double() @ ((q - zeros[:, at // group].double()) * scales[:, at // group].double()).t()
    return (x, codes, scales, zeros), y


UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def far(got, want, dtype):
    """The distance in norm, in units of dtype's rounding."""
    return float((got.double() - want).norm() / want.norm() / UNIT[dtype])
