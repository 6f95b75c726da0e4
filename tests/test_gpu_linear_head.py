"""The appearance head's own layers through the rasteriser: the gradients that a training step takes, against 64 bits."""
import numpy as np
import pytest
import torch  # before anything loads the library: its HIP runtime is the process's

from test_gpu_linear import F32, tb  # noqa: F401
from test_gpu_linear_use import plain

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cells", [0, 7])
def test_a_steps_gradients_through_the_rasteriser(tb, cells):  # noqa: F811
    """Every splat's colour has its own row's offset, and gets its own row's gradient: with cells the rows are sorted on their way."""
    import appearance_head as ah
    import scene
    torch.manual_seed(5)
    sc = scene.make_scene(n=1500, sh_degree=2, width=96, height=64, fx=90.0, seed=3, gt=None)
    view = ah.View(tb, sc, sc.viewmat)
    features = torch.from_numpy(np.concatenate([sc.params[4], sc.params[5]], 1)).to(tb.device)
    where = ah.cells_of(sc.params[0], cells) if cells else None
    assert where is None or not torch.equal(where, where.sort()[0])
    head = ah.AppearanceHead(tb, features.shape[1], 3, hidden=20, embedding=5, dtype=F32, fused=True, cells=where)
    torch.nn.init.normal_(head.leave.weight, std=0.1)
    offset = head(features, 2)
    want, p = plain(head, features, 2, where)
    # a dozen operations of 32 bits with sums of at most 1500 terms: some thousands of units of 2^-24 of the largest value
    assert (offset.cpu().double() - want).abs().max() <= 1e-4 * want.abs().max()
    picture, kept = view.render(offset)
    again, _ = view.render(want.detach().float().to(tb.device))
    # a pixel is a mean of colours with weights that add to at most 1, sums of some hundreds of them in 32 bits
    assert np.abs(picture - again).max() <= 2e-4 * float(want.detach().abs().max()) + 1e-4
    v = view.backward(kept, np.random.default_rng(1).standard_normal(picture.shape).astype(np.float32))
    assert int((v != 0).any(1).sum()) > 500
    offset.backward(v)
    want.backward(v.cpu().double())
    for k, t in head.named_parameters():
        g = p[k].grad
        assert (t.grad.cpu().double() - g).norm() <= 1e-4 * g.norm() + 1e-12, k
