"""The layer norm with several rows to each wave or block, in every width of a row's threads.

Bounds in the 2-norm: a sum over the features is one of at most 16 in a row for each thread, 6 levels
of lanes and 16 waves: 38 roundings, of which y has three sums' and dx two more. A weight's gradient adds
its rows in runs, a block's waves, and the blocks' sums in 32 parts and those: the roundings are
independent of one another, so that n of them in a row are sqrt(n) of 2^-24."""

import pytest
import torch

from delta_ref import F64, HALF, ULP32, close, layer_norm as ref_norm
from tops import _lib
from tops.ops.norm import layer_norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FL = torch.bfloat16, torch.float32


def blocks(D, dt):
    """Blocks that run at once: the partial sums of a call with more rows than they have."""
    return _lib.load().tops_gla_layer_norm_ws_bytes(1 << 24, D, 0 if dt is FL else 1) // (8 * D)


# one wave a row with one, two and four runs a thread (and odd sizes, read one by one); wider ones
@pytest.mark.parametrize("D", [8, 48, 256, 511, 512, 768, 1001, 1024, 1100, 4100, 9000])
@pytest.mark.parametrize("dt", [FL, BF])
def test_more_rows_than_run_at_once(D, dt):
    per = 4 if D <= 1024 else 1
    turns = 2 if D > 1024 else 3
    rows = blocks(D, dt) * per * (turns - 1) + 3 * per + 1   # one turn more for a few blocks
    gen = torch.Generator(device=DEV).manual_seed(D)
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV)   # noqa: E731
    x, dy = r(rows, D).to(dt), r(rows, D).to(dt)
    # every row its own mean and size: another row's would show
    x = (x.float() * (0.5 + torch.rand(rows, 1, generator=gen, device=DEV)) + r(rows, 1)).to(dt)
    d = [t.requires_grad_() for t in (x, 1 + 0.2 * r(D), 0.3 * r(D))]
    y = layer_norm(*d)
    got = torch.autograd.grad(y, d, dy)
    c = [t.detach().to(F64).requires_grad_() for t in d]
    ry = ref_norm(*c)
    want = torch.autograd.grad(ry, c, dy.to(F64))
    own, sums = (HALF if dt is BF else ULP32), 38 ** 0.5 * ULP32
    adds = (turns + 1 + per + blocks(D, dt) / 32 + 32) ** 0.5 * ULP32
    # rows of a mean of up to four times their size lose as much in the differences
    for name, t, w, tol in (("y", y, ry, own + 3 * 4 * sums), ("dx", got[0], want[0], own + 5 * 4 * sums),
                            ("dw", got[1], want[1], 3 * 4 * sums + adds),
                            ("db", got[2], want[2], adds)):
        close(name, t, w.cpu(), tol)
    last = slice(rows - 3 * per - 1, rows)   # the last turn's rows alone
    close("last y", y[last], ry[last].cpu(), own + 3 * 4 * sums)
    close("last dx", got[0][last], want[0][last].cpu(), own + 5 * 4 * sums)
