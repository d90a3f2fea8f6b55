"""GPU: the cases of test_gpu_kv4_sizes.py in calls of many rows."""
import pytest

from test_gpu_kv4 import kv4, torch  # noqa: F401
from test_gpu_kv4_sizes import outweighed, unequal, unseen

pytestmark = pytest.mark.gpu

MANY = [(16, 70, 8, 8, 128, 200), (16, 40, 16, 8, 64, 300), (1, 600, 32, 8, 128, 650)]  # tiles of 128 rows for all SMs


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n,nq,nh,nkv,hd,length", MANY)
def test_unseen_positions_change_nothing(torch, kv4, dtype, n, nq, nh, nkv, hd, length):
    unseen(torch, kv4, dtype, n, nq, nh, nkv, hd, length)


@pytest.mark.parametrize("dtype,apart", [("f16", 16), ("bf16", 16), ("bf16", 26)])
@pytest.mark.parametrize("n,nq,nh,nkv,hd,length", MANY)
def test_blocks_beside_one_another(torch, kv4, dtype, apart, n, nq, nh, nkv, hd, length):
    unequal(torch, kv4, dtype, n, nq, nh, nkv, hd, length, apart)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n,nq,nh,nkv,hd,length", MANY)
def test_positions_of_unequal_values(torch, kv4, dtype, n, nq, nh, nkv, hd, length):
    outweighed(torch, kv4, dtype, n, nq, nh, nkv, hd, length)
