"""LightningIndexer's 8-bit copies of its projections: which copy stands for which weight (the kernels replaced by plain
products, so that a stale copy shows)."""
import copy
import io

import pytest
import torch

from transarch_b200 import indexer_module as M
from transarch_b200._lib import B200DSAError


@pytest.fixture
def mod(monkeypatch):
    monkeypatch.setattr(M.K, "fp8_quantise_blocks", lambda w, scale_fmt=None: (w.clone(), torch.ones(1, 1)))

    def linear(x, codes, scale, *, scale_fmt=None, out_dtype):
        assert x.dim() == 2 and x.stride(1) == 1 and (x.shape[0] < 2 or x.stride(0) >= x.shape[1])
        return (x @ codes.t()).to(out_dtype)

    monkeypatch.setattr(M.K, "fp8_block_linear", linear)
    m = M.LightningIndexer(32, n_heads=2, dtype=torch.float32)
    m.quantise_projections()
    return m


X = torch.randn(3, 32, generator=torch.Generator().manual_seed(0))


def reload(m):
    buf = io.BytesIO()
    torch.save(m, buf)
    buf.seek(0)
    return torch.load(buf, weights_only=False)


@pytest.mark.parametrize("duplicate", [copy.deepcopy, reload])
def test_a_copied_module_keeps_its_copies(mod, duplicate):
    new = duplicate(mod)
    assert torch.equal(new._project("wq", X), mod._project("wq", X))
    # whatever the counters of the new weights say, a changed one is refused, and the original is not concerned
    for _ in range(4):
        with torch.no_grad():
            new.wq.weight.add_(1.0)
        with pytest.raises(B200DSAError, match="wq has changed"):
            new._project("wq", X)
    mod._project("wq", X)
    new._project("wk", X)
    new.quantise_projections()
    assert torch.allclose(new._project("wq", X), X @ new.wq.weight.t())


@pytest.mark.parametrize("duplicate", [copy.deepcopy, reload])
def test_a_stale_copy_stays_stale(mod, duplicate):
    with torch.no_grad():
        mod.wk.weight.mul_(2.0)
    with pytest.raises(B200DSAError, match="wk has changed"):
        duplicate(mod)._project("wk", X)


def test_a_weight_whose_data_was_replaced_is_refused(mod):
    """To another type and back: the counter does not move, the values do."""
    mod.half().float()
    with pytest.raises(B200DSAError, match="wq has changed"):
        mod._project("wq", X)
    mod.quantise_projections()
    mod.wq.half()
    mod.wq.float()
    with pytest.raises(B200DSAError, match="wq has changed"):
        mod._project("wq", X)
    mod._project("wk", X)
    mod.wk.weight.data = mod.wk.weight.data * 2
    with pytest.raises(B200DSAError, match="wk has changed"):
        mod._project("wk", X)
    mod.quantise_projections()
    mod.float()                                                   # nothing to do: nothing is replaced
    assert torch.equal(copy.deepcopy(mod)._project("wk", X), mod._project("wk", X))
    torch.nn.utils.vector_to_parameters(torch.nn.utils.parameters_to_vector(mod.wq.parameters()) + 1, mod.wq.parameters())
    with pytest.raises(B200DSAError, match="wq has changed"):
        copy.deepcopy(mod)._project("wq", X)


@pytest.mark.parametrize("make", [
    lambda x: x.t().contiguous().t(),                             # columns apart
    lambda x: x[:1].expand(3, 32),                                # one row for all tokens
    lambda x: x.view(3, 1, 32),
    lambda x: x.view(3, 2, 16).transpose(1, 2).reshape(3, 32).view(1, 3, 32)[0],
    lambda x: x[:0], lambda x: x[:0].view(0, 1, 32)])
def test_projections_take_what_a_linear_takes(mod, make):
    x = make(X)
    got, want = mod._project("wq", x), mod.wq(x)
    mass = x.abs() @ mod.wq.weight.abs().t()                      # two fp32 sums of 32 products
    assert got.shape == want.shape and bool(((got - want).abs() <= 2 * 32 * 2.0 ** -24 * mass).all())
