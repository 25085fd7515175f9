"""Inputs of 4-bit linears whose every fp32 sum is exact, so that results are compared for equality
(test infrastructure).

Activations are small whole numbers, of one sign in a row, with at least one in every 32 inputs;
scales are powers of two from 2^-2; so each product and sum is a multiple of 2^-2, and exact while it
stays under 2^22 (`Linear.largest`).  Few activations are not zero, so that results are small
and a wrong term is not lost in the one rounding of the result."""
import torch

TERMS = 512  # activations of a row that are not zero, where each 32 inputs need no more than that
LONG_GROUPS = [(2_097_216, 2_097_184), (7_680_256, 1_280_032), (8_388_608, 4_194_336)]  # (K, group)
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
