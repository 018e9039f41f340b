"""Calls of the stand-alone operators that their documentation allows, at the edges: experts that end
inside a warp, outputs in place of inputs, codes at the midpoints, gradients of other types, the
example that the documentation gives."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from litemind_b200 import ops  # noqa: E402
from tests import mx_reference as ref  # noqa: E402

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def same_bits(a, b):
    assert a.shape == b.shape and a.dtype == b.dtype
    kind = {1: torch.uint8, 2: torch.int16, 4: torch.int32}[a.element_size()]
    assert torch.equal(a.contiguous().view(kind), b.contiguous().view(kind))


@pytest.mark.parametrize("experts", [1, 7, 31, 33, 100, 255, 1000, 1023])
def test_sort_plan_over_a_cluster(experts):
    """More pairs than one CTA takes, experts that are no multiple of a warp."""
    idx = torch.randint(-1, experts + 1, (3001, 3), generator=gen(experts), device="cuda", dtype=torch.int32)
    plan = ops.sort_plan(idx, experts)
    offsets, at = ref.sort_plan(idx.cpu(), experts)
    assert torch.equal(plan.offsets.cpu(), offsets) and torch.equal(plan.at.cpu(), at)
