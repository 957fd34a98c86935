"""The operators together, as a network uses them: SC convolutions, a normalised 8-bit head, AdamW steps with the weights
held to their range, and the frozen form."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
def test_training_steps_and_serving(bits):
    import sc_optim
    from sc_layers import LayerNorm, Linear_Int8
    from sc_models import TinyConvSC
    torch.manual_seed(0)
    net = TinyConvSC(classifier="int8", forward="or_2", err=5).cuda()
    assert isinstance(net.fc[0], LayerNorm) and isinstance(net.fc[1], Linear_Int8)
    opt = sc_optim.AdamW(net.parameters(), lr=1e-3, state_bits=bits, clamp=(-1, 0.999))
    x, y = torch.randn(8, 3, 32, 32, device="cuda").clamp(-1, 1), torch.randint(0, 10, (8,), device="cuda")
    for _ in range(3):
        opt.zero_grad(set_to_none=True)
        before = [p.detach().clone() for p in net.parameters()]
        loss = torch.nn.functional.cross_entropy(net(x), y)
        loss.backward()
        assert loss.isfinite() and all(p.grad is not None and p.grad.isfinite().all() for p in net.parameters())
        opt.step()
        for p, b in zip(net.parameters(), before):
            assert p.isfinite().all() and p.min() >= -1 and p.max() <= torch.tensor(0.999) and not torch.equal(p, b)
    net.eval()
    with torch.no_grad():
        want = net(x)
        net.fc[1].freeze()
        assert torch.equal(net(x), want)


def test_resnet18_head():
    from sc_models import ResNet18SC
    torch.manual_seed(0)
    net = ResNet18SC(num_classes=10, classifier="int8", forward="or_2", err=5).cuda()
    x = torch.randn(2, 3, 64, 64, device="cuda")
    net(x).sum().backward()
    assert net.fc[1].weight.grad.shape == (10, 512) and net.fc[0].weight.grad.shape == (512,)


def test_plain_head_is_unchanged():
    from sc_models import ResNet18SC, TinyConvSC
    assert type(TinyConvSC().fc) is torch.nn.Linear and type(ResNet18SC().fc) is torch.nn.Linear
    torch.manual_seed(3)
    a = TinyConvSC()
    torch.manual_seed(3)
    b = TinyConvSC(classifier="float")
    assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))
    with pytest.raises(ValueError, match="classifier"):
        TinyConvSC(classifier="int4")
