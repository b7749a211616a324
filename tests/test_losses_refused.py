"""What the losses over the class axis refuse, before any CUDA call: the C entry points' checks of their arguments, and the
Python operators' on tensors of the wrong kind."""
import pytest
import torch

OK, INVALID, UNSUPPORTED, SCRATCH = 0, -1, -2, -4
P = 4096                                  # a pointer that is never followed


@pytest.fixture(scope="module")
def lib():
    from graph_rws_b200.core import _native
    return _native.lib()


CE = dict(x=P, ldx=8, w=P, ldw=16, order=0, labels=P, label_bytes=8, ignore=-100, rows=4, width=8, classes=16, dtype=0, reduction=1)


def ce_fwd(lib, loss=P, state=P, count=P, scratch=P, scratch_bytes=0, **kw):
    return lib.grws_linear_ce_fwd(*dict(CE, **kw).values(), loss, state, count, scratch, scratch_bytes, None)


def ce_bwd(lib, grad=P, state=P, count=P, dx=P, dw=P, scratch=P, scratch_bytes=0, **kw):
    return lib.grws_linear_ce_bwd(*dict(CE, **kw).values(), grad, state, count, dx, dw, scratch, scratch_bytes, None)


@pytest.mark.parametrize("call", [ce_fwd, ce_bwd])
@pytest.mark.parametrize("status,kw", [
    (INVALID, dict(rows=-1)), (INVALID, dict(width=0)), (INVALID, dict(classes=0)), (INVALID, dict(ldx=7)), (INVALID, dict(ldw=15)),
    (INVALID, dict(order=1, ldw=7)), (INVALID, dict(order=2)), (UNSUPPORTED, dict(dtype=3)), (INVALID, dict(label_bytes=2)),
    (INVALID, dict(reduction=3)), (INVALID, dict(rows=1 << 31)), (INVALID, dict(x=None)), (INVALID, dict(labels=None)), (INVALID, dict(state=None)),
    (INVALID, dict(state=P + 4)), (INVALID, dict(scratch=P + 8)), (INVALID, dict(count=None)), (SCRATCH, dict()),
])
def test_linear_cross_entropy_refuses(lib, call, status, kw):
    assert call(lib, **kw) == status and len(lib.grws_last_error()) > 10


def test_linear_cross_entropy_without_rows_or_gradients(lib):
    assert ce_fwd(lib, rows=0, reduction=0) == OK
    assert ce_bwd(lib, dx=None, dw=None) == OK
    assert lib.grws_linear_ce_scratch_bytes(P, 8, P, 16, 0, 0, 8, 16, 0, 0) == 0


D = dict(z=P, ldz=16, dtype=0, t=P, ldt=4, t_dtype=1, ids=P, ldi=4, id_bytes=8, rows=4, classes=16, kept=4, temperature=2.0, reduction=1)


def distill_fwd(lib, loss=P, state=P, count=P, scratch=P, scratch_bytes=0, **kw):
    return lib.grws_distill_fwd(*dict(D, **kw).values(), loss, state, count, scratch, scratch_bytes, None)


def distill_bwd(lib, grad=P, state=P, count=P, out=P, ldo=16, **kw):
    return lib.grws_distill_bwd(*dict(D, **kw).values(), grad, state, count, out, ldo, None)


@pytest.mark.parametrize("call", [distill_fwd, distill_bwd])
@pytest.mark.parametrize("status,kw", [
    (INVALID, dict(rows=-1)), (INVALID, dict(classes=0)), (INVALID, dict(kept=0)), (UNSUPPORTED, dict(kept=1025, ldt=1025, ldi=1025)), (INVALID, dict(ldz=15)),
    (INVALID, dict(ldt=3)), (INVALID, dict(ldi=3)), (UNSUPPORTED, dict(dtype=-1)), (UNSUPPORTED, dict(t_dtype=3)), (INVALID, dict(id_bytes=1)),
    (INVALID, dict(temperature=0.0)), (INVALID, dict(temperature=-1.0)), (INVALID, dict(temperature=float("nan"))), (INVALID, dict(temperature=float("inf"))),
    (INVALID, dict(reduction=-1)), (INVALID, dict(ldz=1 << 31)), (INVALID, dict(z=None)), (INVALID, dict(t=None)), (INVALID, dict(ids=None)),
    (INVALID, dict(state=None)), (INVALID, dict(state=P + 4)), (INVALID, dict(count=None)),
])
def test_distillation_refuses(lib, call, status, kw):
    assert call(lib, **kw) == status and len(lib.grws_last_error()) > 10


def test_distillation_refuses_short_buffers(lib):
    assert distill_fwd(lib) == SCRATCH
    assert distill_bwd(lib, ldo=15) == INVALID
    assert distill_fwd(lib, rows=0, reduction=0) == OK and distill_bwd(lib, rows=0) == OK


def test_operators_refuse_host_tensors():
    from graph_rws_b200.layers import distillation_loss, linear_cross_entropy
    x, w, y = torch.zeros(4, 8), torch.zeros(8, 16), torch.zeros(4, dtype=torch.long)
    with pytest.raises(RuntimeError, match="CUDA"):
        linear_cross_entropy(x, w, y)
    with pytest.raises(RuntimeError, match="CUDA"):
        distillation_loss(torch.zeros(4, 16), x, y[:, None].expand(4, 8))
    with pytest.raises(ValueError, match="reduction"):
        linear_cross_entropy(x, w, y, reduction="avg")
    with pytest.raises(ValueError, match="reduction"):
        distillation_loss(x, x, y, reduction="batchmean")
