"""GPU: calls of attention and rotary that would lose a derivative are refused."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu

from segquant_b200 import ops

DEV = "cuda"


def _x(*shape, dtype=torch.bfloat16):
    return torch.randn(*shape, device=DEV).to(dtype)


def test_tangents_are_refused(native_lib):
    """Neither operator has a derivative: an input that carries a tangent is refused, not passed on without it."""
    q, pos, w = _x(1, 8, 2, 64), torch.zeros(8, 1, dtype=torch.int32, device=DEV), torch.ones(64, dtype=torch.bfloat16, device=DEV)
    with fwd.dual_level():
        ops.attention(q, q, q)                                   # no tangent: as ever
        ops.rotary(q, q, pos, (64,), norm_q=w, norm_k=w)
        dual = fwd.make_dual(q, torch.ones_like(q))
        dual_w = fwd.make_dual(w, torch.ones_like(w))
        calls = [lambda: ops.attention(dual, q, q), lambda: ops.attention(q, dual, q), lambda: ops.attention(q, q, dual),
                 lambda: ops.rotary(dual, q, pos, (64,)), lambda: ops.rotary(q, dual, pos, (64,)), lambda: ops.rotary(dual, None, pos, (64,)),
                 lambda: ops.rotary(q, q, pos, (64,), norm_q=dual_w, norm_k=w), lambda: ops.rotary(q, q, pos, (64,), norm_q=w, norm_k=dual_w),
                 lambda: ops.rotary(q, q, fwd.make_dual(pos.float(), torch.ones(8, 1, device=DEV)), (64,)), lambda: ops.attention(q, q, q, out=fwd.make_dual(torch.empty_like(q), q)),
                 lambda: ops.rotary(q, q, pos, (64,), out_q=fwd.make_dual(torch.empty_like(q), q))]
        for i, call in enumerate(calls):
            with pytest.raises(RuntimeError, match="no derivative|no backward"):
                call()
                pytest.fail(f"call {i} was not refused")
            with torch.no_grad():                                # reverse mode off does not switch forward mode off
                with pytest.raises(RuntimeError, match="no derivative|no backward"):
                    call()
                    pytest.fail(f"call {i} was not refused without gradients")
        primal = fwd.unpack_dual(dual).primal
        ops.attention(primal, q, q)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: ops.attention(t, q, q), (q,), (torch.ones_like(q),))


def test_gradients_of_positions_are_refused(native_lib):
    q, pos = _x(1, 8, 2, 64), torch.zeros(8, 1, device=DEV, requires_grad=True)
    with pytest.raises(RuntimeError, match="no backward"):
        ops.rotary(q, q, pos, (64,))
    with torch.no_grad():
        ops.rotary(q, q, pos, (64,))
