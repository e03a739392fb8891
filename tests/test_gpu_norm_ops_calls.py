"""Calls of multigrid_amd/norm_ops.py on the GPU that must be refused, or that must return what simpler calls return."""
import pytest
import torch

from multigrid_amd import norm_ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def normal(shape, seed, mean=0.0, std=1.0, dtype=torch.float32):
  g = torch.Generator(device='cuda').manual_seed(seed)
  return torch.empty(shape, device='cuda').normal_(mean, std, generator=g).to(dtype)


def test_clipping_refuses_strided_memory_that_it_would_write_twice():
  """Tensors that go through contiguous copies: their own memory counts, and nothing is written before the refusal."""
  w, q = normal((8, 10), 1), normal((40,), 2)
  for grads, out in (([normal((8, 5), 3), normal((8, 5), 4)], [w[:, :5], w[:, 3:8]]),
                     ([normal((8, 5), 3), w[:, 4:7]], [w[:, :5], torch.zeros(8, 3, device='cuda')]),
                     ([w[::2], w[4:6]], [w[::2], w[4:6]]),
                     ([normal((3, 3), 5)], [q.as_strided((3, 3), (1, 1))]),
                     ([normal((3, 3), 5)], [q.as_strided((3, 3), (2, 1))]),
                     ([normal((4, 2), 5)], [q[:4, None].expand(4, 2)])):
    kept = [t.clone() for t in grads + out]
    with pytest.raises(ValueError, match='overlap'):
      norm_ops.clip_grads(grads, 0.5, out=out)
    assert all(torch.equal(t, k) for t, k in zip(grads + out, kept))


def test_clipping_takes_strided_neighbours():
  w, q = normal((8, 10), 1), normal((24,), 2)
  for parts in ([w[:, :5], w[:, 5:]], [w[::2], w[1::2]], [q[0::3], q[1::3], q[2::3]], [w[:4, :3], w[:4, 3:9], w[4:, 1:]], [w[:, :0], w]):
    norm = torch.sqrt(sum(p.double().square().sum() for p in parts))
    want = [p.double() * torch.clamp(0.5 / (norm + 1e-6), max=1.0) for p in parts]
    got = norm_ops.clip_grads(parts, 0.5, out=parts)[1]
    assert abs(float(got) - float(norm)) <= float(norm) * U * 1.01
    # the factor's two roundings and the product's
    assert all(((p.double() - v).abs() <= v.abs() * (4 * U)).all() for p, v in zip(parts, want))


def test_forward_derivatives_are_refused():
  """The kernels carry no tangents: a dual input, or a dual gradient in the backward pass, raises instead of losing its own."""
  from torch.autograd import forward_ad
  x, w, b = normal((6, 20), 1), normal((20,), 2), normal((20,), 3)
  with forward_ad.dual_level():
    dual = [forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, w, b)]
    for args in ((dual[0], w, b), (x, dual[1], b), (x, w, dual[2]), (x, None, dual[2]), (dual[0].t().contiguous().t(), w, b)):
      with pytest.raises(NotImplementedError, match='forward'):
        norm_ops.layer_norm(*args)
    with pytest.raises(NotImplementedError, match='forward'):
      norm_ops.grad_norm([x, dual[0]])
    with pytest.raises(NotImplementedError, match='forward'):
      norm_ops.clip_grads([x, dual[0]], 0.5)
    wg = w.clone().requires_grad_(True)
    y = norm_ops.layer_norm(x, wg, b)
    with pytest.raises(NotImplementedError, match='forward'):
      torch.autograd.grad(y, wg, forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y)))
    y = norm_ops.layer_norm(x, w, b)      # plain tensors in the same level
    assert forward_ad.unpack_dual(y).tangent is None
  assert torch.equal(norm_ops.layer_norm(x, w, b), y)


def test_recording_a_trace_is_refused():
  """A trace would record the outputs' allocation and not the kernels."""
  from torch.fx.experimental.proxy_tensor import make_fx
  x, w = normal((6, 20), 1), normal((20,), 2)
  calls = (lambda t: norm_ops.layer_norm(t, w), lambda t: norm_ops.grad_norm([t]), lambda t: norm_ops.clip_grads([t], 0.5)[0][0])
  for call in calls:
    with pytest.raises(NotImplementedError, match='trace'):
      torch.jit.trace(call, x, check_trace=False)
    with pytest.raises(NotImplementedError, match='trace'):
      make_fx(call)(x)
    assert torch.isfinite(call(x)).all()
  wg = w.clone().requires_grad_(True)
  y = norm_ops.layer_norm(x, wg)
  with pytest.raises(NotImplementedError, match='trace'):
    make_fx(lambda dy: torch.autograd.grad(y, wg, dy, retain_graph=True)[0])(torch.ones_like(y))
