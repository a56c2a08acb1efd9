"""The layer of experts in README.md: the weighted sum of the experts' rows, run as it stands there."""
import os
import re
from types import SimpleNamespace

import pytest
import torch

README = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "README.md")


def layer_of_the_readme():
    """Its code block, as lines without comments."""
    block, = [b for b in re.findall(r"```python\n(.*?)```", open(README).read(), re.S) if "route_tokens" in b]
    return [line.split("#")[0].rstrip() for line in block.splitlines()]


def test_slots_that_chose_nothing_take_no_row():
    """Rows that belong to nobody are not written by the products and may hold NaN; slots that chose nothing must not bring them in."""
    lines = layer_of_the_readme()
    behind = lines[[i for i, line in enumerate(lines) if line.startswith("down = ")][0] + 1:]
    down = torch.full((8, 3), float("nan"))
    down[:4] = torch.arange(12.0).view(4, 3)
    r = SimpleNamespace(positions=torch.tensor([[0, 2], [-1, -1], [3, -1], [1, -1]], dtype=torch.int32),
                        weights=torch.tensor([[0.25, 0.75], [0.0, 0.0], [1.0, 0.0], [1.0, 0.0]]))
    for nobody in (False, True):
        if nobody:
            r.positions.fill_(-1)
            r.weights.zero_()
            down.fill_(float("nan"))
        names = dict(down=down, r=r, torch=torch)
        exec("\n".join(behind), names)
        want = torch.zeros((4, 3)) if nobody else torch.stack([0.25 * down[0] + 0.75 * down[2], torch.zeros(3), down[3], down[1]])
        assert torch.equal(names["y"], want)


@pytest.mark.gpu
def test_the_layer_runs_as_it_stands(cuda_lib):
    """Tokens of which some have nothing to choose, with NaN left in the memory that the products' results come from."""
    import cutlass_b200 as ops
    T, D, F, E = 40, 64, 48, 4
    g = torch.Generator(device="cuda").manual_seed(1)
    make = lambda *s: torch.randn(s, device="cuda", generator=g).to(torch.bfloat16)  # noqa: E731
    names = dict(ops=ops, torch=torch, T=T, D=D, F=F, E=E, x=make(T, D), w1=make(E, 2 * F, D), w2=make(E, D, F), logits=make(T, E))
    names["logits"][::3] = -float("inf")
    names["logits"][1, 1:] = -float("inf")
    poison = [torch.full((n,), float("nan"), dtype=torch.bfloat16, device="cuda") for n in (2 * T * D, 2 * T * F, 4 * T * F) for _ in range(8)]
    torch.cuda.synchronize()
    del poison
    exec("\n".join(layer_of_the_readme()), names)
    y, r, down = names["y"], names["r"], names["down"]
    assert y.shape == (T, D) and not bool(y[::3].any()) and bool(torch.isfinite(y).all())
    for t in (1, 2, 38):
        want = sum(r.weights[t, j].double() * down[int(r.positions[t, j])].double() for j in range(2) if int(r.positions[t, j]) >= 0)
        assert bool(((y[t].double() - want).abs() <= 2.0 ** -22 * 2 * down.float().nan_to_num().abs().max()).all())
