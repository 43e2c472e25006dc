"""More of what the operators around a served step's linears refuse, on the host."""
import pytest
import torch

from quipsharp_amd.adapters import add_adapters
from quipsharp_amd.rope import append_rotated

BF, I32 = torch.bfloat16, torch.int32


def test_outputs_and_frequencies_that_require_a_gradient_are_refused():
    """A tensor that the call writes would be overwritten behind autograd's back, and learned frequencies lose theirs."""
    grad = lambda *shape, dtype=BF: torch.zeros(*shape, dtype=dtype, requires_grad=True)  # noqa: E731
    z = lambda *shape: torch.zeros(*shape, dtype=BF)  # noqa: E731
    added = lambda outs: add_adapters([z(3, 40)], z(3, 64), torch.zeros(3, dtype=I32), [z(2, 8, 64)], [z(2, 40, 8)],  # noqa: E731
                                      [torch.zeros(2)], outs=outs)
    turned = lambda w, out: append_rotated(z(2, 4, 64), z(2, 2, 64), z(2, 2, 64), z(3, 2, 16, 64), z(3, 2, 16, 64),  # noqa: E731
                                           torch.zeros(2, 3, dtype=I32), torch.zeros(2, dtype=I32), w, out=out)
    ones = torch.ones(32, dtype=torch.float64)
    for call in (lambda: added([grad(3, 40)]), lambda: turned(ones, grad(2, 4, 64)), lambda: turned(grad(32, dtype=torch.float64), None)):
        with pytest.raises(RuntimeError, match="has no gradient"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="runs on the GPU"):
            call()
