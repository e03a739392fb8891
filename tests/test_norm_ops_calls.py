"""Calls of multigrid_amd/norm_ops.py that must be refused or must not change what they return, on the CPU: memory that a
clipping writes twice or reads after writing it, tensors whose graph would end in the call."""
import itertools
import random
import types

import pytest
import torch

from multigrid_amd import norm_ops


def _refused(grads, out):
  """The call is refused, and nothing was written."""
  kept = [t.clone() for t in grads + out]
  with pytest.raises(ValueError, match='overlap|several elements'):
    norm_ops.clip_grads(grads, 0.5, out=out)
  assert all(torch.equal(t, k) for t, k in zip(grads + out, kept))


def test_clipping_refuses_memory_that_it_would_write_twice():
  p, q, w = torch.ones(4), torch.arange(8.0), torch.arange(80.0).reshape(8, 10)
  _refused([p, p], [p, p])
  _refused([q[:4], q[3:]], [q[:4], q[3:]])
  _refused([q[:4], q[4:]], [q[2:6], torch.zeros(4)])      # a result over another tensor's input
  _refused([torch.ones(8, 5), torch.ones(8, 5)], [w[:, :5], w[:, 3:8]])      # column slices that share two columns
  _refused([torch.ones(8, 5), w[:, 4:7]], [w[:, :5], torch.zeros(8, 3)])
  _refused([w[::2], w[4:6]], [w[::2], w[4:6]])
  _refused([torch.ones(3, 3)], [q.as_strided((3, 3), (1, 1))])      # windows: one tensor with an element at two places
  _refused([torch.ones(3, 3)], [q.as_strided((3, 3), (2, 1))])
  _refused([torch.ones(4, 2)], [torch.zeros(4, 1).expand(4, 2)])
  a = torch.nn.Parameter(torch.zeros(4))
  a.grad = torch.ones(4)
  with pytest.raises(ValueError):
    norm_ops.clip_grad_norm_([a, a], 0.5)
  assert torch.equal(a.grad, torch.ones(4))


def _clipped(grads, norm_of=None):
  norm = torch.sqrt(sum(g.double().square().sum() for g in grads))
  return [(g.double() * min(1.0, 0.5 / (float(norm) + 1e-6))).float() for g in grads], norm


def test_clipping_takes_neighbours_that_share_no_element():
  """Interleaved views: column slices, every other row, the two halves of a complex-like layout; inputs that overlap while the
  results lie apart; a result over its own gradient in another order."""
  w, q = torch.randn(8, 10), torch.randn(24)
  for parts in ([w[:, :5], w[:, 5:]], [w[::2], w[1::2]], [q[0::2], q[1::2]], [q[0::3], q[1::3], q[2::3]], [w[:4, :3], w[:4, 3:9], w[4:, 1:]],
                [w.t()[:4], w.t()[4:]], [q.as_strided((2, 2), (3, 2)), q.as_strided((2,), (5,), 1)], [w[:, :0], w]):
    want, norm = _clipped(parts)
    got = norm_ops.clip_grads(parts, 0.5, out=parts)[1]
    assert torch.allclose(got.double(), norm) and all(torch.allclose(p, v, rtol=1e-6) for p, v in zip(parts, want))
  want, _ = _clipped([q[:9], q[3:12]])
  got, _ = norm_ops.clip_grads([q[:9], q[3:12]], 0.5, out=[torch.zeros(9), torch.zeros(9)])
  assert all(torch.allclose(p, v, rtol=1e-6) for p, v in zip(got, want))
  s = torch.randn(6, 6)
  want, _ = _clipped([s.clone()])
  assert torch.allclose(norm_ops.clip_grads([s], 0.5, out=[s.t()])[0][0], want[0], rtol=1e-6)
  meta = torch.zeros(4, device='meta')      # no memory at all
  assert norm_ops.clip_grads([meta, meta], 0.5, out=[meta, meta])[1].is_meta


def test_overlap_is_told_exactly():
  """Small random views of one buffer: refused if and only if an address is written twice, or written for one tensor and
  read for another."""
  rng = random.Random(5)
  seen = {True: 0, False: 0}
  for _ in range(3000):
    base = torch.zeros(64)
    views, places = [], []
    for _ in range(2):
      dims = rng.randint(1, 3)
      shape = [rng.randint(1, 4) for _ in range(dims)]
      stride = [rng.choice((1, 2, 3, 4, 5, 7, 8)) for _ in range(dims)]
      reach = sum((n - 1) * s for n, s in zip(shape, stride))
      if reach >= 64:
        shape, reach = [1] * dims, 0
      at = rng.randint(0, 63 - reach)
      views.append(base.as_strided(shape, stride, at))
      places.append([at + sum(i * s for i, s in zip(index, stride)) for index in itertools.product(*(range(n) for n in shape))])
    written, other = places
    bad = len(set(written)) < len(written) or bool(set(written) & set(other))
    seen[bad] += 1
    grads, out = [torch.ones(views[0].shape), views[1]], [views[0], torch.zeros(views[1].shape)]
    if bad:
      _refused(grads, out)
    else:
      norm_ops.clip_grads(grads, 0.5, out=out)
  assert min(seen.values()) > 300


def test_no_graph_is_cut_without_a_word():
  """A norm, or results apart, of tensors that carry a graph would be constants to autograd."""
  leaf = torch.ones(4, requires_grad=True)
  for g in (leaf, leaf * 2):
    with pytest.raises(RuntimeError, match='no derivative'):
      norm_ops.grad_norm([torch.ones(3), g])
    with pytest.raises(RuntimeError, match='no derivative'):
      norm_ops.clip_grads([torch.ones(3), g], 0.5)
    with torch.no_grad():
      assert float(norm_ops.grad_norm(g)) == float(g.norm()) and len(norm_ops.clip_grads([g], 0.5)[0]) == 1
    assert float(norm_ops.grad_norm([g.detach()])) == float(g.norm())
  # in place and into given memory: outside autograd, as torch.nn.utils.clip_grad_norm_ is
  p = torch.nn.Parameter(torch.ones(4))
  p.square().sum().backward(create_graph=True)
  assert p.grad.requires_grad and float(norm_ops.clip_grad_norm_([p], 0.5)) == 4.0
  out = torch.zeros(4)
  norm_ops.clip_grads([leaf * 2], 0.5, out=[out])
  assert not out.requires_grad and torch.allclose(out, torch.full((4,), 0.25))


def test_the_kernels_take_one_device():
  """What the policies' clipping asks before it calls the kernels: a policy over several devices is left to torch."""
  def grad(device='cuda:0', **kw):
    return types.SimpleNamespace(**{'is_cuda': True, 'device': torch.device(device), 'dtype': torch.float32, 'layout': torch.strided, **kw})
  assert norm_ops.takes([grad(), grad(dtype=torch.bfloat16)]) and norm_ops.takes([grad('cuda:1'), grad('cuda:1')])
  assert not norm_ops.takes([grad(), grad('cuda:1')]) and not norm_ops.takes([]) and not norm_ops.takes([torch.ones(3)])
  assert not norm_ops.takes([grad(), grad(dtype=torch.float64)]) and not norm_ops.takes([grad(layout=torch.sparse_coo)])


def test_fake_tensors_have_no_memory_to_overlap():
  from torch._subclasses.fake_tensor import FakeTensorMode
  with FakeTensorMode():
    grads = [torch.ones(4), torch.ones(3, 3).t(), torch.ones(4)]
    out, norm = norm_ops.clip_grads(grads, 0.5, out=grads)
    assert norm.shape == () and [o.shape for o in out] == [g.shape for g in grads]
    assert norm_ops.layer_norm(torch.ones(3, 4)).shape == (3, 4) and norm_ops.grad_norm(grads, 0).shape == ()
