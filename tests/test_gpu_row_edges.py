"""Row operators (elg_amd/logits.py) at the edges of what their documentation allows, against the definitions in 64 bits (row_oracle.py)."""
import numpy as np
import pytest
import torch

import row_oracle as ro

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def lg():
    from elg_amd import logits
    return logits


def rng(seed):
    return torch.Generator(device="cpu").manual_seed(seed)


def host(t):
    return t.detach().cpu().double().numpy()


# ------------------------------------------------------------------------------------------------------------- top_logits
@pytest.mark.parametrize("V,k,dtype", [(2049, 1, "float32"), (3001, 64, "float32"), (5003, 256, "bfloat16"), (20001, 256, "float16"),
                                       (65536, 100, "float32"), (70001, 256, "float32"), (131075, 128, "bfloat16")])
def test_top_of_rows_with_thousands_of_nan(V, k, dtype):
    """A diverged policy's rows: all NaN, all but one, more NaN than candidates fit and fewer open nodes than k beside them.  The lowest
    indices of the NaN come first, then the best of the others."""
    g = rng(V)
    z = torch.randn(12, V, generator=g).to(TYPES[dtype])
    z[0] = float("nan")
    z[1, :-1] = float("nan")
    z[2, torch.randperm(V, generator=g)[:1100]] = float("nan")
    z[3, torch.randperm(V, generator=g)[:V - 7]] = float("nan")
    z[4] = torch.where(torch.arange(V) % 2 == 0, float("nan"), -np.inf)
    z[5, :max(1, k // 2)] = float("nan")
    z[6:9] = z[0]
    z[9, 1::2] = -float("nan")
    rv, ri = ro.top(host(z), k)
    for _ in range(3):
        values, idx, tail = lg().top_logits(z.to(DEV), k, with_tail=True)
        np.testing.assert_array_equal(idx.cpu().numpy(), ri)
        np.testing.assert_array_equal(host(values), rv)
        assert torch.isnan(tail[:10]).all() and torch.isfinite(tail[10:]).all()
