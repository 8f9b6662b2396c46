"""SiftLM.loss takes the targets that forward takes."""
import pytest
import torch

from swiftx_b200.sift import SiftConfig, SiftLM

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("shape", [(150,), (150, 1), (6, 25)])
def test_loss_of_reshaped_targets(shape):
    """forward flattens its targets; so does loss(): the same values and gradients whatever their shape."""
    torch.manual_seed(0)
    model = SiftLM(SiftConfig(vocab_size=300, d_model=64, n_layers=1)).to(DEV)
    idx, tgt = torch.randint(0, 300, (3, 50), device=DEV), torch.randint(0, 300, (3, 50), device=DEV)
    got = []
    for y in (tgt, tgt.reshape(shape)):
        model.zero_grad()
        loss = model.loss(idx, y)
        loss.backward()
        got.append([loss.detach()] + [p.grad.clone() for p in model.parameters()])
    for a, b in zip(*got):
        assert torch.equal(a, b)
    # fp32 products on either side: off by a few d 2^-24 of logits below 1 (weights of 0.02)
    assert abs(float(got[0][0]) - float(model(idx, tgt.reshape(shape))[1])) <= 2.0 ** -16 * float(got[0][0])
    with pytest.raises(ValueError):
        model.loss(idx, tgt[:2])
