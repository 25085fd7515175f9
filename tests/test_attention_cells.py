"""What attention_cells.py's inputs tell apart: keys left out of the definition, on the CPU."""
import pytest
import torch

import attention_cells as cells
from test_gpu_attention_cells import PAGED, WINDOW

CASES = sorted({(max(lengths), reps, dim, dtype) for lengths, reps, _, dim, _, dtype, _, _, _ in PAGED}
               | {(keys, reps, dim, dtype) for _, _, keys, reps, _, dim, dtype, _, _ in WINDOW})


@pytest.mark.parametrize("run", [1, 32, 700, 5000])
@pytest.mark.parametrize("n,reps,dim,dtype", CASES)
def test_tiles_left_out(n, reps, dim, dtype, run):
    """The results miss the bound without the first, the last or any run of 32 keys between them."""
    dtype = {"bf16": torch.bfloat16, "f16": torch.float16}[dtype]
    see = torch.ones(n, dtype=torch.bool)
    want = cells.shares(cells.counts(see, reps, dim, run))
    cells.check(want.to(dtype), want, dtype)
    tiles = -(-n // 32)
    for i in {0, tiles - 1, *range(0, tiles, max(1, tiles // 60))}:
        less = see.clone()
        less[i * 32:i * 32 + 32] = False
        if bool(less.any()):
            with pytest.raises(AssertionError):
                cells.check(cells.shares(cells.counts(less, reps, dim, run)).to(dtype), want, dtype)


def test_against_the_definition():
    for n, reps, dim, run in ((70, 3, 64, 5), (333, 16, 64, 1), (40, 5, 96, 32), (1, 4, 64, 32)):
        k, v = cells.keys_values(n, reps, dim, run, 4.0)
        p = torch.softmax(cells.queries(reps, dim).double() @ k.double().t(), -1)
        want = cells.shares(cells.counts(torch.ones(n, dtype=torch.bool), reps, dim, run), 4.0)
        assert bool(((p @ v.double() - want).abs() < 1e-20 + 1e-12 * want).all())
