"""GPU suite of the quantised KV cache at its edges: scores, lists and arguments at the ends of what the
calls take, against the definitions in 64 bits (tests/kv_reference.py)."""
import numpy as np
import pytest
import torch

from tests.test_gpu_kv import dev, kv, make  # noqa: F401  (kv: a fixture)

pytestmark = pytest.mark.gpu


# ---- lists -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("past", [0, 1, 20])
@pytest.mark.parametrize("path", [[-2, -1], [-5, -3], [-1, 0], [-2 ** 31, -2 ** 31 + 1], [-3, 2], [0, 2 ** 31 - 1], [-2 ** 31, 3]])
def test_paths_below_zero_are_reported_and_move_nothing(kv, hf, past, path):
    from huffman_amd import HuffhipError
    ctx = hf.Context()
    c = make(kv, "e4m3", 4, 16, 2, 64, 32, ctx=ctx)
    g = torch.Generator(device="cuda").manual_seed(2)
    for pool in (c.k, c.v):
        pool.copy_(torch.randint(0, 0x70, pool.shape, generator=g, device="cuda", dtype=torch.uint8))
    before = [t.clone() for t in (c.k, c.v, c.k_scale, c.v_scale)]
    table, cu = dev(np.array([[3, 1], [2, 0]], np.int32)), dev(np.array([0, 4, 8], np.int32))
    kv_len = np.array([past + 4, past + 4], np.int32)
    torch.cuda.synchronize()
    new_len = c.keep(table, dev(kv_len), cu, dev(np.array([path, [0, 1]], np.int32)), dev(np.array([2, 2], np.int32)))
    with pytest.raises(HuffhipError):
        ctx.sync()
    assert new_len.tolist() == [past + 4, past + 2]  # (the other sequence's path stays where it is)
    for t, was in zip((c.k, c.v, c.k_scale, c.v_scale), before):
        assert torch.equal(t, was)
