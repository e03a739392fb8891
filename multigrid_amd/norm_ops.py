"""torch bindings of include/mgrid_norm.h: layer norm with its gradients, and clipping by the global gradient norm, both in
the trainer's stacked form too (every tensor with a leading agent axis, one weight row and one norm per agent).

`layer_norm(x, weight, bias)` is what the policies call with `layer_norm=True`; `clip_grad_norm_` is the clipping of an update
epoch (v8_robust_ppo.py:340).  `clip_grads` is the same clipping into other tensors, `grad_norm` the norm alone.  On a GPU
they run the HIP kernels of libmgnn.so on the current stream, for float32, bfloat16 and float16 (a missing library raises);
CPU tensors take the plain torch expression of the same formulas.  What neither takes is refused with a TypeError (types,
layouts) or a ValueError (shapes, sizes, devices, overlapping memory) before anything is written.

Nothing is kept between calls: workspaces come from torch's allocator, so every captured graph has its own.
"""
import array
import ctypes as C
import functools
import math
import operator

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from . import fused_ops

MAX_COLS = 16384      # MGNN_LN_MAX_C
MAX_GROUPS = 65535    # MGNN_MAX_GROUPS
TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}

# name -> (restype, argtypes): every symbol include/mgrid_norm.h declares
SYMBOLS = {
    'mgnn_layer_norm': (C.c_int, [C.c_void_p, C.c_int64] + [C.c_void_p] * 4 + [C.c_int64, C.c_int64, C.c_int, C.c_double, C.c_int, C.c_int,
                                                                            C.c_void_p]),
    'mgnn_layer_norm_workspace': (C.c_int64, [C.c_int64, C.c_int64, C.c_int, C.c_int]),
    'mgnn_layer_norm_backward': (C.c_int, [C.c_void_p, C.c_int64] + [C.c_void_p] * 7 + [C.c_int64, C.c_int64, C.c_int64, C.c_int, C.c_int,
                                                                                     C.c_int, C.c_void_p]),
    'mgnn_grad_norm_workspace': (C.c_int64, [C.c_void_p, C.c_void_p, C.c_int64, C.c_int64]),
    'mgnn_grad_norm': (C.c_int, [C.c_void_p] * 3 + [C.c_int64, C.c_int64, C.c_void_p, C.c_void_p, C.c_int64, C.c_void_p]),
    'mgnn_clip_grads': (C.c_int, [C.c_void_p] * 4 + [C.c_int64, C.c_int64, C.c_double, C.c_void_p, C.c_void_p, C.c_int64, C.c_void_p]),
}
ERRORS = {1: 'a size is out of range', 2: 'the kernel launch failed', 3: 'an element type is not supported', 4: 'the workspace does not fit',
          5: 'an argument is invalid', 6: 'a gradient that is written overlaps another one'}
_LIB = None


def load():
  global _LIB
  if _LIB is None:
    fused_ops.load()      # raises if libmgnn.so is missing
    lib = C.CDLL(fused_ops.LIB_PATH)
    for name, (res, args) in SYMBOLS.items():
      fn = getattr(lib, name)
      fn.restype, fn.argtypes = res, args
    _LIB = lib
  return _LIB


def _call(fn, dev, *args):
  """fn(*args, stream) on dev, whose current stream it enqueues on."""
  stream = torch._C._cuda_getCurrentRawStream(dev.index)
  if torch.cuda.current_device() == dev.index:
    rc = fn(*args, stream)
  else:
    with torch.cuda.device(dev):
      rc = fn(*args, stream)
  if rc != 0:
    raise (RuntimeError if rc == 2 else ValueError)('%s: %s (MGNN error %d)' % (fn.__name__, ERRORS.get(rc, 'unknown'), rc))


# ---- layer norm ----

def _ln_args(x, weight, bias, eps):
  """The number of weight rows (1, or the leading axis of x)."""
  if x.dtype not in TYPES or x.layout is not torch.strided:
    raise TypeError('layer_norm takes dense float32, bfloat16 or float16 tensors, not %s' % x.dtype)
  if x.dim() < 1 or not 1 <= x.size(-1) <= MAX_COLS:
    raise ValueError('layer_norm takes rows of 1 to %d elements, not a tensor of shape %s' % (MAX_COLS, tuple(x.shape)))
  if not 0 <= eps < math.inf:
    raise ValueError('layer_norm takes a finite eps >= 0, not %r' % (eps,))
  groups = 1
  for t in (weight, bias):
    if t is None:
      continue
    if t.dtype not in (x.dtype, torch.float32) or t.layout is not torch.strided:
      raise TypeError("layer_norm's weight and bias are of x's type (%s) or float32, not %s" % (x.dtype, t.dtype))
    if t.device != x.device:
      raise ValueError("layer_norm's weight and bias are on %s, x on %s" % (t.device, x.device))
    shape = t.shape
    if len(shape) == 2 and x.dim() >= 2 and shape[0] == x.size(0):
      groups = shape[0]
    elif len(shape) != 1:
      shape = ()
    if not shape or shape[-1] != x.size(-1):
      raise ValueError("layer_norm's weight or bias of shape %s does not fit x of shape %s: [cols] or [x.shape[0], cols] is wanted"
                       % (tuple(t.shape), tuple(x.shape)))
  if weight is not None and bias is not None and (weight.dtype != bias.dtype or weight.shape != bias.shape):
    raise ValueError("layer_norm's weight and bias differ in shape or type")
  if groups > MAX_GROUPS:
    raise ValueError('layer_norm takes at most %d weight rows, not %d' % (MAX_GROUPS, groups))
  return groups


def _rows(x, cols):
  """x with its rows contiguous and at one distance (x itself or a view of it where that holds), and that distance."""
  if x.is_contiguous():
    return x, cols
  x = x.reshape(-1, cols)
  if (cols > 1 and x.stride(1) != 1) or (x.shape[0] > 1 and x.stride(0) < cols):
    return x.contiguous(), cols
  return x, x.stride(0) if x.shape[0] > 1 else cols


@functools.lru_cache(maxsize=1024)
def _workspace(groups, rows, cols, kind):
  return load().mgnn_layer_norm_workspace(groups, rows, cols, kind)


def _ln_forward(x, weight, bias, eps, groups, want_stats):
  """y, and what the backward pass takes of the call: x by rows, its row distance, the statistics, the weight, the sizes."""
  cols = x.shape[-1]
  n = x.numel() // cols
  x2, ld = _rows(x, cols)
  y = torch.empty_like(x) if x2 is x else torch.empty(x.shape, dtype=x.dtype, device=x.device)
  w = b = None
  kind = wkind = TYPES[x.dtype]
  if weight is not None:
    w = weight.contiguous()
    wkind = TYPES[w.dtype]
  if bias is not None:
    b = bias.contiguous()
    wkind = TYPES[b.dtype]
  stats = torch.empty(2 * n, dtype=torch.float32, device=x.device) if want_stats else None
  sizes = (groups, n // groups if groups else 0, cols)
  _call(load().mgnn_layer_norm, x.device, x2.data_ptr(), ld, w.data_ptr() if weight is not None else None,
        b.data_ptr() if bias is not None else None, y.data_ptr(), stats.data_ptr() if want_stats else None, *sizes, eps, kind, wkind)
  return y, x2, ld, stats, w, sizes, (kind, wkind)


def _ln_backward(ctx, dy):
  x, stats, w = ctx.saved_tensors
  ld, sizes, kinds, bias = ctx.plan
  want_x, want_w, want_b = ctx.needs_input_grad[:3]
  dev = x.device
  dy = dy.contiguous()
  dx = torch.empty_like(dy) if want_x else None
  dw = torch.empty_like(w) if want_w else None
  db = (torch.empty_like(w) if w is not None else torch.empty(bias[0], dtype=bias[1], device=dev)) if want_b else None
  size = _workspace(*sizes, kinds[0]) if want_w or want_b else 0
  room = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
  _call(load().mgnn_layer_norm_backward, dev, x.data_ptr(), ld, dy.data_ptr(), w.data_ptr() if w is not None else None, stats.data_ptr(),
        dx.data_ptr() if want_x else None, dw.data_ptr() if want_w else None, db.data_ptr() if want_b else None,
        room.data_ptr() if size else None, size, *sizes, *kinds)
  return dx, dw, db, None, None


_ln_backward_once = once_differentiable(_ln_backward)


class _LayerNorm(torch.autograd.Function):

  @staticmethod
  def forward(ctx, x, weight, bias, eps, groups):
    y, x2, ld, stats, w, sizes, kinds = _ln_forward(x, weight, bias, eps, groups, True)
    ctx.save_for_backward(x2, stats, w)
    ctx.plan = (ld, sizes, kinds, (bias.shape, bias.dtype) if weight is None and bias is not None else None)
    return y

  @staticmethod
  def backward(ctx, dy):
    # grad mode is on in here only under create_graph: then a second backward pass has to be refused
    return _ln_backward_once(ctx, dy) if torch.is_grad_enabled() else _ln_backward(ctx, dy)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
  """Layer norm over the last axis: (x - mean) / sqrt(mean((x - mean)^2) + eps) * weight + bias, in x's type, with the
  statistics and every sum in float32.  weight / bias: [cols] of x's type or float32, or None; [x.shape[0], cols] gives
  every index of x's leading axis (an agent) its own.  Rows of 1 to 16384 elements.  Differentiable once in all three."""
  groups = _ln_args(x, weight, bias, eps)
  if x.is_cuda:
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
      return _LayerNorm.apply(x, weight, bias, eps, groups)
    return _ln_forward(x, weight, bias, eps, groups, False)[0]
  h = F.layer_norm(x.float(), x.shape[-1:], None, None, eps)
  wide = (x.shape[0],) + (1,) * (x.dim() - 2) + x.shape[-1:]      # a stacked weight against x
  if weight is not None:
    h = h * (weight.float().reshape(wide) if weight.dim() == 2 else weight.float())
  if bias is not None:
    h = h + (bias.float().reshape(wide) if bias.dim() == 2 else bias.float())
  return h.to(x.dtype)


# ---- the global gradient norm ----

def _dense(t, stacked):
  """Whether t's elements fill one stretch of memory, in whatever order (stacked: agent by agent)."""
  if t.is_contiguous():
    return True
  order = sorted(range(t.dim()), key=lambda d: (t.stride(d), d == 0), reverse=True)
  return t.permute(order).is_contiguous() and (not stacked or order[0] == 0)


def _grad_list(grads, stacked):
  grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
  if not isinstance(stacked, int) or not 0 <= stacked <= MAX_GROUPS:
    raise ValueError('stacked is the length of the leading agent axis, 0 (none) to %d, not %r' % (MAX_GROUPS, stacked))
  dev = grads[0].device if grads else None
  for kind in {(g.dtype, g.layout) for g in grads}:
    if kind[0] not in TYPES or kind[1] is not torch.strided:
      raise TypeError('gradients are dense float32, bfloat16 or float16 tensors, not %s, %s' % kind)
  if len({g.device for g in grads}) > 1:
    raise ValueError('gradients are on several devices: %s' % ', '.join(sorted({str(g.device) for g in grads})))
  if stacked:
    for g in grads:
      if g.dim() < 1 or g.size(0) != stacked:
        raise ValueError('a gradient of shape %s has no leading agent axis of %d' % (tuple(g.shape), stacked))
  return grads, dev


def takes(grads):
  """Whether grads, a list, are what the kernels take: tensors on a GPU, of the types they know."""
  return bool(grads) and all(g.is_cuda and g.dtype in TYPES and g.layout is torch.strided for g in grads)


def _launch(src, dst, max_norm, stacked, dev):
  """The kernels on dense tensors; dst None: the norms alone."""
  lib, groups, count = load(), stacked or 1, len(src)
  n = array.array('q', [t.numel() // groups for t in src] if stacked else [t.numel() for t in src])
  types = array.array('i', [TYPES[t.dtype] for t in src])
  sp = array.array('Q', [t.data_ptr() for t in src])
  norms = torch.empty((stacked,) if stacked else (), dtype=torch.float32, device=dev)
  np, tp = n.buffer_info()[0], types.buffer_info()[0]
  size = lib.mgnn_grad_norm_workspace(np, tp, count, groups)
  room = torch.empty(size, dtype=torch.uint8, device=dev) if size > 0 else None
  work = room.data_ptr() if size > 0 else None
  if dst is None:
    _call(lib.mgnn_grad_norm, dev, sp.buffer_info()[0], np, tp, count, groups, norms.data_ptr(), work, size)
  else:
    dp = sp if dst is src else array.array('Q', [t.data_ptr() for t in dst])
    _call(lib.mgnn_clip_grads, dev, sp.buffer_info()[0], dp.buffer_info()[0], np, tp, count, groups, max_norm, norms.data_ptr(), work, size)
  return norms


def _plain_norms(grads, stacked):
  if not grads:
    return torch.zeros((stacked,) if stacked else ())
  sq = sum(g.double().reshape(stacked or 1, -1).square().sum(dim=1) for g in grads)
  return sq.sqrt() if stacked else sq.sqrt()[0]


@torch.no_grad()
def grad_norm(grads, stacked=0):
  """The 2-norm of all gradients together, a float32 scalar on their device; stacked=A: every gradient has a leading
  agent axis of A, and agent a's norm is element a of the result.  Squares are added in float64.  No gradients: 0."""
  grads, dev = _grad_list(grads, stacked)
  if dev is None or dev.type != 'cuda':
    return _plain_norms(grads, stacked).float()
  return _launch([g if _dense(g, stacked) else g.contiguous() for g in grads], None, 0.0, stacked, dev)


@torch.no_grad()
def clip_grads(grads, max_norm, stacked=0, out=None):
  """([g * min(1, max_norm / (norm + 1e-6)) for every gradient g], norm) with norm = grad_norm(grads, stacked); agent by
  agent if stacked.  out: tensors of the gradients' shapes and types that receive the results (the gradients themselves:
  in place); none of them may overlap another gradient of the call.  A norm that is NaN makes every result NaN."""
  grads, dev = _grad_list(grads, stacked)
  max_norm = float(max_norm)
  if not max_norm >= 0:
    raise ValueError('max_norm is a number >= 0, not %r' % max_norm)
  plain = all([g.is_contiguous() for g in grads])      # every tensor of the call
  if out is None:
    out = [torch.empty_like(g) for g in grads]
  else:
    out = list(out)
    apart = len(out) != len(grads) or not all(map(operator.is_, out, grads))
    if apart and ([o.shape for o in out] != [g.shape for g in grads] or [o.dtype for o in out] != [g.dtype for g in grads]
                  or any([o.device != dev for o in out])):
      raise ValueError('out does not match the gradients in number, shape, type or device')
    plain = plain and (not apart or all([o.is_contiguous() for o in out]))
    if not plain and any(0 in [s for s, k in zip(o.stride(), o.shape) if k > 1] for o in out):
      raise ValueError('a gradient that is written has several elements at one address (an expanded tensor)')
  if dev is None or dev.type != 'cuda':
    norms = _plain_norms(grads, stacked)
    factor = (max_norm / (norms + 1e-6)).clamp(max=1.0).float()
    for o, g in zip(out, grads):
      o.copy_(g.float() * factor.reshape(factor.shape + (1,) * (g.dim() - factor.dim())))
    return out, norms.float()
  src, dst = grads, out
  if not plain:
    src, dst = [], []
    for g, o in zip(grads, out):
      if (g.is_contiguous() and o.is_contiguous()) or (g.stride() == o.stride() and _dense(g, stacked)):
        src.append(g)
        dst.append(o)
      else:      # no common dense order: through contiguous copies
        src.append(g.contiguous())
        dst.append(torch.empty(o.shape, dtype=o.dtype, device=dev))
  norms = _launch(src, dst, max_norm, stacked, dev)
  torch.autograd.graph.increment_version(dst)      # written behind autograd's back: a graph that saved one of them will say so
  if not plain:
    for d, o in zip(dst, out):
      if d is not o:
        o.copy_(d)
  return out, norms


def clip_grad_norm_(parameters, max_norm, stacked=0):
  """torch.nn.utils.clip_grad_norm_ (v8_robust_ppo.py:340) on the parameters' .grad in place; parameters without one are
  left out.  stacked=A: agent by agent.  Returns the norm(s) before clipping."""
  parameters = [parameters] if isinstance(parameters, torch.Tensor) else parameters
  grads = [p.grad for p in parameters if p.grad is not None]
  return clip_grads(grads, max_norm, stacked, out=grads)[1]
