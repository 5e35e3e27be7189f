"""graphslim_amd.ops record no graph: a tensor whose gradient would be lost is refused.  No GPU."""
import pytest
import torch

W, IDS, TI, V = torch.zeros(3, 4), torch.zeros(3, dtype=torch.int32), torch.zeros(3, 1, dtype=torch.int32), torch.zeros(3)


def calls(ops, p):
    """Every entry point with p in each place that autograd would reach."""
    return [lambda: ops.embedding(p, IDS), lambda: ops.embedding(W, IDS, out=p), lambda: ops.embedding_grad(p, IDS, 3),
            lambda: ops.gated_ffn(p, W, W), lambda: ops.gated_ffn(W, p, W), lambda: ops.gated_ffn(W, W, p),
            lambda: ops.gated_ffn_grad(p, W, W, W, W), lambda: ops.gated_ffn_grad(W, p, W, W, W), lambda: ops.distill(p, W[:, :1], TI),
            lambda: ops.distill(W, p[:, :1], TI), lambda: ops.distill_grad(p, W[:, :1], TI, V, V), lambda: ops.distill_loss_grad(p, W[:, :1], TI, V)]


def test_tensors_that_require_a_gradient(monkeypatch):
    from graphslim_amd import ops
    p = torch.zeros(3, 4, requires_grad=True)
    real = ops._device

    def on_gpu(**tensors):                               # as if all of them were on a GPU: only what comes before is looked at
        try:
            return real(**tensors)
        except ValueError as e:
            if "no CPU path" not in str(e):
                raise
            for t in tensors.values():
                if t.requires_grad and torch.is_grad_enabled():
                    return real(**{"first": t})
            return torch.device("cpu")
    monkeypatch.setattr(ops, "_device", on_gpu)
    monkeypatch.setattr(ops._lib, "lib", lambda: (_ for _ in ()).throw(AssertionError("reached")))
    for call in calls(ops, p):
        with pytest.raises(ValueError, match="requires a gradient"):
            call()


def test_without_recording_they_are_taken():
    from graphslim_amd import ops
    p = torch.zeros(3, 4, requires_grad=True)
    with torch.no_grad():
        for call in calls(ops, p):
            with pytest.raises(ValueError, match="no CPU path"):
                call()
    for call in calls(ops, p.detach()):
        with pytest.raises(ValueError, match="no CPU path"):
            call()
