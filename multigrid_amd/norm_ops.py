"""Layer norm with its gradients, and clipping by the global gradient norm (include/mgrid_norm.h), both in the trainer's
stacked form too: every tensor with a leading agent axis, one weight row and one norm per agent.

`layer_norm(x, weight, bias)` is what the policies call with `layer_norm=True`; `clip_grad_norm_` is the clipping of an update
epoch (v8_robust_ppo.py:340).  `clip_grads` is the same clipping into other tensors, `grad_norm` the norm alone.  On a GPU
they run the HIP kernels of libmgnn.so on the current stream, for float32, bfloat16 and float16; other tensors take the
plain torch expression of the same formulas.  The checks, the autograd node and the memory are csrc/norm_torch.cpp, built as
_norm_ops.so; a missing library raises.  What is not taken is refused with a TypeError (types, layouts) or a ValueError
(shapes, sizes, devices, overlapping memory) before anything is written; what would lose its derivative, with a RuntimeError
(NotImplementedError for forward-mode tangents, which the kernels do not carry, and while torch.jit.trace or make_fx
records, which would not see the kernels).

Nothing is kept between calls: workspaces come from torch's allocator, so every captured graph has its own.  As with any
torch operator, a backward pass that is captured needs leaves whose eager graphs are gone.
"""
import importlib.util
import os

import torch

from . import fused_ops

EXT_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), '_norm_ops.so')
MAX_COLS = 16384      # MGNN_LN_MAX_C
MAX_GROUPS = 65535    # MGNN_MAX_GROUPS
TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}      # MGNN_F32, MGNN_BF16, MGNN_F16
_EXT = None


def load():
  """The extension module over libmgnn.so."""
  global _EXT
  if _EXT is None:
    fused_ops.load()      # raises if libmgnn.so is missing
    if not os.path.exists(EXT_PATH):
      raise ImportError('multigrid_amd: %s is missing. Build it with `python -c "import __graft_entry__ as g; g.build()"`.' % EXT_PATH)
    spec = importlib.util.spec_from_file_location('multigrid_amd._norm_ops', EXT_PATH)
    ext = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ext)
    _EXT = ext
  return _EXT


def layer_norm(x, weight=None, bias=None, eps=1e-5):
  """Layer norm over the last axis: (x - mean) / sqrt(mean((x - mean)^2) + eps) * weight + bias, in x's type, with the
  statistics and every sum in float32.  weight / bias: [cols] of x's type or float32, or None; [x.shape[0], cols] gives
  every index of x's leading axis (an agent) its own.  Rows of 1 to 16384 elements.  Differentiable in all three, once: on
  a GPU its gradients have no graph, and asking for one (create_graph) raises, as a forward-mode tangent does."""
  return (_EXT or load()).layer_norm(x, weight, bias, eps)


def grad_norm(grads, stacked=0):
  """The 2-norm of all gradients together, a float32 scalar on their device; stacked=A: every gradient has a leading
  agent axis of A, and agent a's norm is element a of the result.  Squares are added in float64.  No gradients: 0.
  It has no derivative: tensors that require grad are refused unless grad mode is off."""
  return (_EXT or load()).grad_norm([grads] if isinstance(grads, torch.Tensor) else list(grads), stacked)


def clip_grads(grads, max_norm, stacked=0, out=None):
  """([g * min(1, max_norm / (norm + 1e-6)) for every gradient g], norm) with norm = grad_norm(grads, stacked); agent by
  agent if stacked.  out: tensors of the gradients' shapes and types that receive the results, each its gradient itself (in
  place) or other memory; none of them may overlap itself, another result or another gradient of the call.  A norm that is
  NaN makes every result NaN.  It has no derivative: without out, tensors that require grad are refused unless grad mode is
  off; out is written outside autograd, whatever graph the gradients carry."""
  return (_EXT or load()).clip_grads([grads] if isinstance(grads, torch.Tensor) else list(grads), max_norm, stacked,
                                     out if out is None else list(out))


def clip_grad_norm_(parameters, max_norm, stacked=0):
  """torch.nn.utils.clip_grad_norm_ (v8_robust_ppo.py:340) on the parameters' .grad in place; parameters without one are
  left out.  stacked=A: agent by agent.  Returns the norm(s) before clipping.  Outside autograd, as torch's is."""
  parameters = [parameters] if isinstance(parameters, torch.Tensor) else parameters
  grads = [p.grad for p in parameters if p.grad is not None]
  return (_EXT or load()).clip_grads(grads, max_norm, stacked, grads)[1]


def takes(grads):
  """Whether grads, a list, are what the kernels take: tensors on one GPU, of the types they know."""
  return bool(grads) and all(g.is_cuda and g.device == grads[0].device and g.dtype in TYPES and g.layout is torch.strided for g in grads)
