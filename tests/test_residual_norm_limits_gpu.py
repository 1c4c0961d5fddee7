"""The residual norm at the far ends of the sizes it takes."""
import pytest
import torch

from jirf_hip import train_ops as T

pytestmark = pytest.mark.gpu


def test_parameter_gradients_of_the_most_images():
    """2^31 - 1 images of one token and one channel: the last worker's images end past 31 bits unless counted in 64.  All but
    the first and the last two images are zero, so each gradient is a sum of three small whole numbers, exact in any order;
    with mean 0 and reciprocal deviation 1 as the statistics, vh is y."""
    B = 2**31 - 1
    at = torch.tensor([0, B - 2, B - 1], device="cuda")
    dn, y = (torch.zeros(B, 1, 1, dtype=torch.float16, device="cuda") for _ in range(2))
    dn[at, 0, 0] = torch.tensor([1.0, 2.0, 4.0], dtype=torch.float16, device="cuda")
    y[at, 0, 0] = torch.tensor([3.0, 5.0, 7.0], dtype=torch.float16, device="cuda")
    stats = torch.zeros(4, B, 1, device="cuda")
    stats[3] = 1.0
    pre = (1, torch.ones(1, device="cuda"), torch.zeros(1, device="cuda"))
    g = T.residual_norm_bwd(None, dn, y, None, stats, pre=pre, scale=None, layout="tokens")
    assert float(g["dpre_b"]) == 1 + 2 + 4
    assert float(g["dpre_w"]) == 1 * 3 + 2 * 5 + 4 * 7
