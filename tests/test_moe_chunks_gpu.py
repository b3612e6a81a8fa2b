"""w4_moe_route's order by expert where the last chunk of tokens holds one or a few tokens."""
import pytest
import torch

from xe2x2_b200 import ops

pytestmark = pytest.mark.gpu


def _sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


# chunks of 16 tokens up to 16 for each SM, then equal shares of the SMs, at most 1024
@pytest.mark.parametrize("tokens", [lambda n: 33, lambda n: 49, lambda n: 16 * n - 15, lambda n: 16 * n + 1,
                                    lambda n: 17 * (n - 1) + 1, lambda n: 1024 * n + 1,
                                    lambda n: 1024 * (n + 3) + 1])
@pytest.mark.parametrize("E,k", [(32, 4), (300, 3)])
def test_a_last_chunk_of_few_tokens(cuda, tokens, E, k):
    T = tokens(_sms())
    x = torch.randn(T, E, generator=torch.Generator(device="cuda").manual_seed(T), device=cuda)
    x[-1], x[T // 2] = torch.arange(E, device=cuda) * 0.01, -float("inf")  # the last token's own choice; padding
    r = ops.moe_route(x, k)
    ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
    ids[T // 2] = E  # nowhere
    assert r.ids[-1].tolist() == list(range(E - 1, E - 1 - k, -1))
    assert torch.equal(torch.where(r.ids < 0, E, r.ids).long(), ids)
    flat = ids.reshape(-1)
    order = torch.sort(flat, stable=True).indices
    live = T * k - k
    assert torch.equal(r.rows[:live].long(), order[:live] // k) and (r.rows[live:] == -1).all()
    back = torch.empty_like(order)
    back[order] = torch.arange(T * k, device=cuda)
    back[flat == E] = -1
    assert torch.equal(r.slots.long().reshape(-1), back)
    assert torch.equal(r.offsets[1:].long(), torch.cumsum(torch.bincount(flat, minlength=E + 1)[:E], 0))
