"""Serving operators at the ends of their ranges."""
import pytest
import torch

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


# ------------------------------------------------------------------------------------------- token log probabilities
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,V,top", [(3, 4, 4), (2, 32, 32), (3, 700, 20), (400, 700, 3), (1000, 200, 2), (1, 200000, 32), (2, 200000, 1)])
def test_nan_in_the_first_column_is_the_first_alternative(dtype, N, V, top):
    """NaN is above +inf and the lowest index comes first: ids in order whatever column it lies in, the first slice's or a later
    slice's first among them (rows of 200000 columns are split over a cluster)."""
    from hydra_b200.sampling import token_logprobs
    x = torch.randn(N, V, generator=torch.Generator().manual_seed(V)).to(dtype)
    x[:, 0] = NAN
    x[-1, V // 2], x[-1, V - 1] = NAN, INF
    r = token_logprobs(x.cuda(), torch.ones(N, dtype=torch.int64).cuda(), top=top)
    key = x.float().nan_to_num(nan=INF, posinf=3e38)
    assert torch.equal(r.top_ids.cpu(), torch.sort(key, dim=1, descending=True, stable=True).indices[:, :top])
    assert r.logprobs.isnan().all() and r.entropy.isnan().all() and r.top_logprobs.isnan().all()
