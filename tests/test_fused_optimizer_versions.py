"""A step of torch's fused optimizers is seen by the network: the packed weights and the flat
parameter conduit go by the parameters' versions, which those optimizers do not advance by themselves."""
import pytest
import torch

from v2e2v_amd import CistaLSTCNet


@pytest.mark.parametrize("kind", [torch.optim.Adam, torch.optim.AdamW, torch.optim.SGD])
def test_fused_step_advances_the_versions(kind):
    model = CistaLSTCNet([16, 16], base_channels=32, depth=2, num_bins=5)
    params = list(model.parameters())
    for p in params[1:]:
        p.grad = torch.ones_like(p)
    opt = kind(params, lr=0.1, fused=True)
    before = [p._version for p in params]
    opt.step()
    assert params[0]._version == before[0]                  # no gradient: not written
    assert all(p._version > v for p, v in zip(params[1:], before[1:]))


@pytest.mark.gpu
def test_network_uses_the_weights_of_a_fused_step():
    torch.manual_seed(0)
    model = CistaLSTCNet([16, 16], base_channels=32, depth=2, num_bins=5).to("cuda").train()
    x, prev = torch.randn(1, 5, 16, 16, device="cuda"), torch.zeros(1, 1, 16, 16, device="cuda")
    opt = torch.optim.Adam(model.parameters(), lr=1e-2, fused=True)
    out, _ = model(x, prev, None)
    out.mean().backward()
    opt.step()
    twin = CistaLSTCNet([16, 16], base_channels=32, depth=2, num_bins=5).to("cuda")
    twin.load_state_dict(model.state_dict())
    with torch.no_grad():
        new = model(x, prev, None)[0]
        assert torch.equal(new, twin(x, prev, None)[0]) and not torch.equal(new, out.detach())
