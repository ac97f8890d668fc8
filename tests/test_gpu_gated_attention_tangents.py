"""Forward-mode derivatives: the operators have none, and say so instead of dropping a tangent."""
import pytest
import torch
import torch.autograd.forward_ad as fw

pytestmark = pytest.mark.gpu


def test_a_tangent_is_refused():
    from tracklab_amd import attention as A
    from tracklab_amd._lib import TlkError
    g = torch.Generator().manual_seed(1)
    rnd = lambda *s: torch.randn(*s, generator=g).cuda()      # noqa: E731
    q, k, v, u, tab = rnd(1, 5, 2, 16), rnd(1, 5, 2, 16), rnd(1, 5, 2, 16), rnd(1, 5, 2, 16), rnd(3, 2)
    buckets = torch.tensor([0, 1, 2], dtype=torch.int32).cuda()
    args = {"q": q, "k": k, "v": v, "gate": u, "bias": tab}
    h, x, w = rnd(3, 32), rnd(3, 32), rnd(32)
    joint = {"h": h, "residual": x, "weight": w, "bias": w, "gate": h, "res_scale": w, "next_weight": w, "next_bias": w}
    with fw.dual_level():
        want = A.gated_attention(buckets=buckets, **args)      # (a level alone changes nothing)
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                for n in args:
                    with pytest.raises(TlkError, match="forward-mode"):
                        A.gated_attention(buckets=buckets, **{**args, n: fw.make_dual(args[n], torch.ones_like(args[n]))})
                for n in joint:
                    with pytest.raises(TlkError, match="forward-mode"):
                        A.norm_gate_residual(norm="layer", next_norm="layer", **{**joint, n: fw.make_dual(joint[n], torch.ones_like(joint[n]))})
    assert torch.equal(want, A.gated_attention(buckets=buckets, **args))
