"""Heads of 256 on both sides of the rule for who makes the plan, against the definition in 64 bits."""
import pytest

from test_gpu_shared_attention import Pool, same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("common", [2200, 2500, 2900, 3800])
@pytest.mark.parametrize("dtype,cache", [("bf16", "bf16"), ("f16", "e4m3")])
def test_large_heads(common, dtype, cache, hip):
    same(Pool([(common, [100, 1, 57, 0])], 40, 8, 256, 16, dtype, cache, seed=common))


@pytest.mark.parametrize("common", [300, 500])
def test_large_heads_of_many_sequences(common, hip):
    same(Pool([(common, [30 + i for i in range(12)])], 24, 24, 256, 16, seed=common))
