"""Operators for training a student on a teacher's top logits, on rows in fp32, fp16 or bf16 (csrc/gs_embedding.hip, gs_gated.hip,
gs_distill.hip; the C entry points are in include/gslim.h):

    embedding, embedding_grad                  rows of a table by token / node id, scaled; the table's gradient
    gated_ffn, gated_ffn_grad                  h = act(x Wg^T) * (x Wu^T) and its backward pass
    distill, distill_grad, distill_loss_grad   tau^2 KL(teacher's top logits || student) per row and its gradient

Gradients are explicit calls, like everywhere in this package: no autograd, and a tensor that requires a gradient is refused while autograd
records, since its gradient would be lost in silence.  Every call runs on the current stream of its tensors'
device (which need not be the current device) and takes its outputs and scratch from torch's allocator there, so it can be captured
into a graph, and calls on two streams or in two graphs share nothing.  A tensor that another stream writes or frees has to be
synchronised by the caller, as for any torch call.  Matrices may have any row stride; their rows have to be dense.  An `out` that lies
on another operand is refused, but for distill_*'s on the whole of the logits.
"""
from __future__ import annotations

import math

import torch

from . import _lib
from ._lib import check

_raw_stream = torch._C._cuda_getCurrentRawStream      # the handle of torch.cuda.current_stream(device), without an object around it

TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
ACTIVATIONS = {"silu": 0, "gelu": 1, "relu": 2, "sigmoid": 3}
MAX_TOP = 1024


def _refuse(message):
    raise ValueError(f"graphslim_amd.ops: {message}")


def _device(**tensors):
    """The one GPU all of them are on."""
    dev = None
    for name, t in tensors.items():
        if not isinstance(t, torch.Tensor):
            _refuse(f"{name} is a tensor (got {type(t).__name__})")
        if t.requires_grad and torch.is_grad_enabled():
            _refuse(f"{name} requires a gradient, which these calls do not record: call them under torch.no_grad(), or with {name}.detach()")
        if dev is None:
            dev = t.device
            if dev.type != "cuda":
                _refuse(f"{name} is on {dev}: there is no CPU path")
        elif t.device != dev:
            _refuse(f"{name} is on {t.device}, other arguments on {dev}")
    return dev


def _matrix(name, t, cols=None, rows=None, dtype=None):
    """Row stride of a 2-D tensor with dense rows."""
    if t.dim() != 2:
        _refuse(f"{name} has two dimensions (got {tuple(t.shape)})")
    n, c = t.shape
    ld, step = t.stride()
    if dtype is not None and t.dtype != dtype:
        _refuse(f"{name} is {t.dtype}, other arguments {dtype}")
    if t.dtype not in TYPES:
        _refuse(f"{name} is fp32, fp16 or bf16 (got {t.dtype})")
    if cols is not None and c != cols:
        _refuse(f"{name} has {c} columns, {cols} are wanted")
    if rows is not None and n != rows:
        _refuse(f"{name} has {n} rows, {rows} are wanted")
    if c == 0:
        _refuse(f"{name} has no columns")
    if step != 1 and c > 1:
        _refuse(f"the rows of {name} are not dense (strides {(ld, step)})")
    if n <= 1:
        return c
    if ld < c:
        _refuse(f"the rows of {name} overlap (strides {(ld, step)})")
    return ld


def _vector(name, t, n, dtype):
    if t.dtype != dtype:
        _refuse(f"{name} is {dtype} (got {t.dtype})")
    if not (tuple(t.shape) == (n,) and t.is_contiguous()):
        _refuse(f"{name} is a dense vector of {n} (got {tuple(t.shape)}, strides {t.stride()})")


def _apart(out, ld, **inputs):
    """Refuses an `out` (row stride ld) that lies on an input: inputs are tensors, dense ones, or (matrix, row stride)."""
    def span(t, ld=None):
        e = t.element_size()
        return (t.data_ptr(), t.shape[0], ld * e, t.shape[1] * e) if ld is not None else (t.data_ptr(), 1, t.numel() * e, t.numel() * e)
    p, n, s, c = span(out, ld)
    for name, t in inputs.items():
        q, m, r, d = span(*t) if isinstance(t, tuple) else span(t)
        if not (n and m and c and d) or q >= p + (n - 1) * s + c or p >= q + (m - 1) * r + d:
            continue
        if (n == 1) != (m == 1) or (n > 1 and s == r):      # columns of one matrix side by side lie apart
            step = s if n > 1 else r
            if c <= (q - p) % step <= step - d:
                continue
        _refuse(f"out lies on {name}")


def _ids(ids):
    if ids.dtype != torch.int32:
        _refuse(f"ids are int32 (got {ids.dtype})")
    if not ids.is_contiguous():
        _refuse(f"ids are dense (strides {ids.stride()})")


def _scratch(nbytes, dev):
    return torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes > 0 else None


def _ptr(t):
    return None if t is None else t.data_ptr()


def _launch(dev, call, *args):
    """call(*args, stream) on the current stream of `dev`, with that device the current one."""
    if dev.index == torch.cuda.current_device():
        rc = call(*args, _raw_stream(dev.index))
    else:
        with torch.cuda.device(dev):
            rc = call(*args, _raw_stream(dev.index))
    if rc:
        check(rc)


# ------------------------------------------------------------------------------------------------
# embedding
# ------------------------------------------------------------------------------------------------


def embedding(table, ids, scale=1.0, out=None):
    """scale * table[ids], of shape ids.shape + (width,); an id outside the table is padding and gives zeros.  `out`: a
    [ids.numel(), width] matrix that receives the rows and is returned as it is."""
    dev = _device(table=table, ids=ids)
    ld = _matrix("table", table)
    if table.shape[0] <= 0:
        _refuse("table has no rows")
    _ids(ids)
    n, F = ids.numel(), table.shape[1]
    if out is None:
        out = torch.empty(*ids.shape, F, dtype=table.dtype, device=dev)
        ldo = F
    else:
        _device(table=table, out=out)
        ldo = _matrix("out", out, F, n, table.dtype)
        _apart(out, ldo, table=(table, ld), ids=ids)
    _launch(dev, _lib.lib().gs_embedding_fwd, table.data_ptr(), ld, table.shape[0], F, TYPES[table.dtype], ids.data_ptr(), n, scale,
            out.data_ptr(), ldo)
    return out


def embedding_grad(d_out, ids, n_rows, scale=1.0, out=None, accumulate=False, dtype=None):
    """Gradient [n_rows, width] of `embedding`'s table: scale times the sum of d_out's rows of each id.  The sum is
    one of partial sums of consecutive tokens, cut where the ids and the sizes say: two runs are bitwise equal.  d_out: ids.shape +
    (width,), or [ids.numel(), width] with any row stride.  dtype: that of d_out (default) or torch.float32.  `out` receives the gradient;
    with accumulate=True it is added to what `out` holds."""
    dev = _device(d_out=d_out, ids=ids)
    _ids(ids)
    n = ids.numel()
    if d_out.dim() != 2:
        if not (d_out.dim() >= 1 and tuple(d_out.shape[:-1]) == tuple(ids.shape)):
            _refuse(f"d_out is {tuple(d_out.shape)}, ids are {tuple(ids.shape)}")
        if not d_out.is_contiguous():
            _refuse(f"d_out is dense, or a matrix (strides {d_out.stride()})")
        d_out = d_out.view(n, d_out.shape[-1])
    ldd = _matrix("d_out", d_out, rows=n)
    n_rows, F = int(n_rows), d_out.shape[1]
    if n_rows <= 0:
        _refuse(f"a table of {n_rows} rows")
    given = out is not None
    if not given:
        if accumulate:
            _refuse("accumulate=True adds to `out`, which is missing")
        dtype = d_out.dtype if dtype is None else dtype
        if dtype not in (d_out.dtype, torch.float32):
            _refuse(f"the gradient is {d_out.dtype} or torch.float32 (got {dtype})")
        out = torch.empty(n_rows, F, dtype=dtype, device=dev)
    else:
        _device(d_out=d_out, out=out)
        if dtype not in (None, out.dtype):
            _refuse(f"out is {out.dtype}, dtype {dtype}")
        if out.dtype not in (d_out.dtype, torch.float32):
            _refuse(f"the gradient is {d_out.dtype} or torch.float32 (got {out.dtype})")
    ldw = _matrix("out", out, F, n_rows)
    if given:
        _apart(out, ldw, d_out=(d_out, ldd), ids=ids)
    L = _lib.lib()
    scratch = _scratch(L.gs_embedding_bwd_scratch_bytes(n, n_rows, F), dev)
    _launch(dev, L.gs_embedding_bwd, d_out.data_ptr(), ldd, TYPES[d_out.dtype], ids.data_ptr(), n, n_rows, F, scale, bool(accumulate),
            out.data_ptr(), ldw, TYPES[out.dtype], _ptr(scratch))
    return out


# ------------------------------------------------------------------------------------------------
# gated feed-forward block
# ------------------------------------------------------------------------------------------------


def _gated_args(x, w_gate, w_up, act):
    if act not in ACTIVATIONS:
        _refuse(f"act is one of {', '.join(ACTIVATIONS)} (got {act!r})")
    dev = _device(x=x, w_gate=w_gate, w_up=w_up)
    ldx = _matrix("x", x)
    M, D = x.shape
    ldw = _matrix("w_gate", w_gate, D, dtype=x.dtype)
    F = w_gate.shape[0]
    if F <= 0:
        _refuse("w_gate has no rows")
    ldu = _matrix("w_up", w_up, D, F, x.dtype)
    if ldw != ldu:
        _refuse(f"w_gate and w_up have one row stride (got {ldw} and {ldu})")
    return dev, ldx, ldw, M, D, F


def _plain(ldx, ldw, D, *matrices):
    """Whether rows of D elements consist of whole, aligned chunks of 16 bytes (the library asks it of 16-bit types)."""
    return (D | ldx | ldw) % 8 == 0 and not any(t.data_ptr() % 16 for t in matrices)


def gated_ffn(x, w_gate, w_up, act="silu", save=False):
    """act(x w_gate^T) * (x w_up^T) for x [M, D] and w_gate, w_up [F, D].  save=True returns (h, saved): `saved` holds the two
    projections, [2, M, F] in fp32, for `gated_ffn_grad`."""
    dev, ldx, ldw, M, D, F = _gated_args(x, w_gate, w_up, act)
    h = torch.empty(M, F, dtype=x.dtype, device=dev)
    saved = torch.empty(2, M, F, dtype=torch.float32, device=dev) if save else None
    L = _lib.lib()
    scratch = _scratch(L.gs_gated_fwd_scratch_bytes(M, D, F, TYPES[x.dtype], _plain(ldx, ldw, D, x, w_gate, w_up)), dev)
    _launch(dev, L.gs_gated_fwd, x.data_ptr(), ldx, w_gate.data_ptr(), w_up.data_ptr(), ldw, TYPES[x.dtype], M, D, F, ACTIVATIONS[act],
            h.data_ptr(), F, _ptr(saved), _ptr(scratch))
    return (h, saved) if save else h


def gated_ffn_grad(d_h, x, w_gate, w_up, saved, act="silu"):
    """(d_x, d_w_gate, d_w_up) of `gated_ffn` for the gradient d_h [M, F] of its result; `saved` as the forward call gave it."""
    dev, ldx, ldw, M, D, F = _gated_args(x, w_gate, w_up, act)
    _device(x=x, d_h=d_h, saved=saved)
    lddh = _matrix("d_h", d_h, F, M, x.dtype)
    if not (saved.dtype == torch.float32 and tuple(saved.shape) == (2, M, F) and saved.is_contiguous()):
        _refuse(f"saved is what gated_ffn(save=True) gave: [2, {M}, {F}] in fp32 (got {saved.dtype}, {tuple(saved.shape)}, strides {saved.stride()})")
    d_x = torch.empty(M, D, dtype=x.dtype, device=dev)
    d_wg, d_wu = (torch.empty(F, D, dtype=x.dtype, device=dev) for _ in range(2))
    L = _lib.lib()
    scratch = _scratch(L.gs_gated_bwd_scratch_bytes(M, D, F, TYPES[x.dtype], _plain(ldx, ldw, D, x, w_gate, w_up)), dev)
    _launch(dev, L.gs_gated_bwd, d_h.data_ptr(), lddh, x.data_ptr(), ldx, w_gate.data_ptr(), w_up.data_ptr(), ldw, saved.data_ptr(),
            TYPES[x.dtype], M, D, F, ACTIVATIONS[act], d_x.data_ptr(), D, d_wg.data_ptr(), d_wu.data_ptr(), D, _ptr(scratch))
    return d_x, d_wg, d_wu


# ------------------------------------------------------------------------------------------------
# distillation
# ------------------------------------------------------------------------------------------------


def _distill_args(logits, top_values, top_ids, tau):
    dev = _device(logits=logits, top_values=top_values, top_ids=top_ids)
    ldz = _matrix("logits", logits)
    n, V = logits.shape
    if not (top_values.dim() == 2 and top_values.shape[0] == n and top_values.is_contiguous()):
        _refuse(f"top_values are dense, one row a row of logits (got {tuple(top_values.shape)}, strides {top_values.stride()})")
    if top_values.dtype != logits.dtype:
        _refuse(f"top_values are {top_values.dtype}, logits {logits.dtype}")
    k = top_values.shape[1]
    if not (1 <= k <= MAX_TOP):
        _refuse(f"1 to {MAX_TOP} teacher entries a row (got {k})")
    if tuple(top_ids.shape) != (n, k):
        _refuse(f"top_ids are {tuple(top_ids.shape)}, top_values {(n, k)}")
    _ids(top_ids)
    tau = float(tau)
    if not (0 < tau <= torch.finfo(torch.float32).max and math.log2(math.e) / tau < torch.finfo(torch.float32).max):   # what fp32 holds
        _refuse(f"a temperature of {tau}")
    return dev, (logits.data_ptr(), ldz, TYPES[logits.dtype], n, V, top_values.data_ptr(), top_ids.data_ptr(), k, tau), n


def _grad_out(logits, out, ldz, **inputs):
    if out is None:
        return torch.empty(logits.shape, dtype=logits.dtype, device=logits.device), logits.shape[1]
    _device(logits=logits, out=out)
    ld = _matrix("out", out, logits.shape[1], logits.shape[0], logits.dtype)
    if out.data_ptr() != logits.data_ptr() or ld != ldz:
        inputs["logits"] = logits, ldz
    _apart(out, ld, **inputs)
    return out, ld


def distill(logits, top_values, top_ids, tau=1.0):
    """(loss, lse), one fp32 value a row: loss = tau^2 KL(p || q) with p the softmax of the teacher's top logits / tau over the
    row's entries and q that of logits / tau over all classes; lse = log sum exp(logits / tau), which `distill_grad` takes.
    An entry whose class (top_ids) is none of the logits', or whose value is -inf, is not there; a row without any has loss 0."""
    dev, args, n = _distill_args(logits, top_values, top_ids, tau)
    loss, lse = (torch.empty(n, dtype=torch.float32, device=dev) for _ in range(2))
    _launch(dev, _lib.lib().gs_distill_fwd, *args, loss.data_ptr(), lse.data_ptr())
    return loss, lse


def distill_grad(logits, top_values, top_ids, lse, d_loss, tau=1.0, out=None):
    """Gradient of sum(d_loss * loss) with respect to the logits, in their type; rows with d_loss 0 or without teacher entries get 0.
    out=logits overwrites them."""
    dev, args, n = _distill_args(logits, top_values, top_ids, tau)
    _device(logits=logits, lse=lse, d_loss=d_loss)
    _vector("lse", lse, n, torch.float32)
    _vector("d_loss", d_loss, n, torch.float32)
    out, ldd = _grad_out(logits, out, args[1], top_values=top_values, top_ids=top_ids, lse=lse, d_loss=d_loss)
    _launch(dev, _lib.lib().gs_distill_bwd, *args, lse.data_ptr(), d_loss.data_ptr(), out.data_ptr(), ldd)
    return out


def distill_loss_grad(logits, top_values, top_ids, d_loss, tau=1.0, out=None):
    """(loss, gradient) in one call, for row weights d_loss that are known beforehand (1 / n for a mean): the logits are read once
    where a row fits the registers of a workgroup."""
    dev, args, n = _distill_args(logits, top_values, top_ids, tau)
    _device(logits=logits, d_loss=d_loss)
    _vector("d_loss", d_loss, n, torch.float32)
    out, ldd = _grad_out(logits, out, args[1], top_values=top_values, top_ids=top_ids, d_loss=d_loss)
    loss = torch.empty(n, dtype=torch.float32, device=dev)
    _launch(dev, _lib.lib().gs_distill_loss_grad, *args, d_loss.data_ptr(), loss.data_ptr(), out.data_ptr(), ldd)
    return loss, out
