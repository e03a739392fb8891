"""multigrid_amd/norm_ops.py without a GPU: the C ABI against include/mgrid_norm.h, every refusal (they come before any
launch), and the plain expressions that CPU tensors take."""
import array
import ctypes as C
import os
import re

import pytest
import torch

import norm_abi
from multigrid_amd import norm_ops, ppo

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _header():
  return re.sub(r'/\*.*?\*/', '', open(os.path.join(ROOT, 'include', 'mgrid_norm.h')).read(), flags=re.S)


def test_every_declared_symbol_is_exported_and_bound():
  src = _header()
  names = sorted(set(re.findall(r'\b(mgnn_[a-z_0-9]+)\s*\(', src)))
  assert sorted(norm_abi.SYMBOLS) == names
  lib = norm_abi.load()
  assert all(hasattr(lib, n) for n in names)
  define = dict(re.findall(r'#define (\w+) (\d+)', src))
  assert int(define['MGNN_LN_MAX_C']) == norm_ops.MAX_COLS and int(define['MGNN_MAX_GROUPS']) == norm_ops.MAX_GROUPS
  assert [int(define[n]) for n in ('MGNN_F32', 'MGNN_BF16', 'MGNN_F16')] == list(norm_ops.TYPES.values())


def _list(ns, types):
  n, t = array.array('q', ns), array.array('i', types)
  return n, t, n.buffer_info()[0], t.buffer_info()[0]


def test_layer_norm_entry_points_refuse_before_any_launch():
  lib = norm_abi.load()
  shape, typ, ws, val = 1, 3, 4, 5
  one = C.c_void_p(16)      # never dereferenced: refused first

  def fwd(ld=8, groups=1, rows=4, cols=8, eps=1e-5, t=0, w=0, x=one, y=one):
    return lib.mgnn_layer_norm(x, ld, None, None, y, None, groups, rows, cols, eps, t, w, None)
  assert fwd(cols=0, ld=8) == shape and fwd(cols=norm_ops.MAX_COLS + 1, ld=1 << 20) == shape and fwd(ld=7) == shape
  assert fwd(groups=-1) == shape and fwd(rows=-1) == shape and fwd(groups=norm_ops.MAX_GROUPS + 1) == shape
  assert fwd(rows=1 << 61) == shape
  assert fwd(t=3) == typ and fwd(t=-1) == typ and fwd(t=0, w=1) == typ and fwd(t=1, w=2) == typ
  assert fwd(eps=-1.0) == val and fwd(eps=float('nan')) == val and fwd(x=None) == val and fwd(y=None) == val
  assert fwd(rows=0) == 0 and fwd(groups=0) == 0 and fwd(rows=0, x=None, y=None) == 0

  def bwd(ld=8, groups=1, rows=100000, cols=8, t=0, w=0, stats=one, room=None, size=0, dw=one):
    return lib.mgnn_layer_norm_backward(one, ld, one, None, stats, one, dw, None, room, size, groups, rows, cols, t, w, None)
  need = lib.mgnn_layer_norm_workspace(1, 100000, 8, 0)
  assert need > 0 and lib.mgnn_layer_norm_workspace(1, 1, 8, 0) == 0 and lib.mgnn_layer_norm_workspace(0, 1, 8, 0) == 0
  assert lib.mgnn_layer_norm_workspace(1, 1, 0, 0) == -1 and lib.mgnn_layer_norm_workspace(1, 1, 8, 9) == -1
  assert bwd() == ws and bwd(room=one, size=need - 1) == ws and bwd(room=C.c_void_p(20), size=need) == ws
  assert bwd(stats=None) == val and bwd(ld=1) == shape and bwd(w=1) == typ
  assert bwd(groups=0) == 0
  assert lib.mgnn_layer_norm_backward(one, 8, one, None, one, None, None, None, None, 0, 1, 4, 8, 0, 0, None) == 0      # nothing wanted
  assert lib.mgnn_layer_norm_backward(one, 8, one, None, one, one, None, None, None, 0, 1, 0, 8, 0, 0, None) == 0      # no rows


def test_gradient_entry_points_refuse_before_any_launch():
  lib = norm_abi.load()
  shape, typ, ws, val, over = 1, 3, 4, 5, 6
  one = C.c_void_p(16)

  def call(ns, types, src, dst, groups=1, max_norm=1.0, norms=one, room=None, size=0):
    # a large tensor far away joins every list, so that each needs a workspace, which is asked for last and never given
    ns, types, src, dst = ns + [1 << 22], types + [0], src + [1 << 40], dst + [1 << 40]
    n, t, np_, tp = _list(ns, types)
    s, d = array.array('Q', src), array.array('Q', dst)
    return lib.mgnn_clip_grads(s.buffer_info()[0], d.buffer_info()[0], np_, tp, len(ns), groups, max_norm, norms, room, size, None)
  assert call([4], [7], [64], [64]) == typ
  assert call([-1], [0], [64], [64]) == shape and call([4], [0], [64], [64], groups=0) == shape
  assert call([4], [0], [64], [64], groups=norm_ops.MAX_GROUPS + 1) == shape and call([1 << 61], [0], [64], [64], groups=8) == shape
  assert call([4], [0], [64], [64], max_norm=-1.0) == val and call([4], [0], [64], [64], max_norm=float('nan')) == val
  assert call([4], [0], [0], [64]) == val and call([4], [0], [64], [0]) == val and call([4], [0], [64], [64], norms=None) == val
  assert call([4], [0], [64], [64]) == ws and call([4], [0], [64], [64], room=C.c_void_p(12), size=1 << 20) == ws
  # 4 floats at 64 are 64..80: the same memory twice, a partial overlap, a result over another tensor's input
  assert call([4, 4], [0, 0], [64, 64], [64, 64]) == over and call([4, 4], [0, 0], [64, 76], [64, 76]) == over
  assert call([4, 4], [0, 0], [64, 128], [256, 72]) == over and call([4], [0], [64], [68]) == over
  assert call([4, 4], [0, 0], [64, 64], [128, 136]) == over
  assert call([4, 2], [0, 0], [64, 96], [64, 96], groups=3) == over      # 3 groups of 4 floats reach 112
  # neighbours, an empty tensor inside another, and one input read twice are no overlap (the workspace is what is missing)
  assert call([4, 4], [0, 0], [64, 80], [64, 80]) == ws and call([4, 0], [0, 0], [64, 64], [64, 64]) == ws
  assert call([4, 4], [0, 0], [64, 64], [128, 144]) == ws
  n, t, np_, tp = _list([4, 5000, 0], [0, 1, 2])
  assert lib.mgnn_grad_norm_workspace(np_, tp, 3, 2) % 8 == 0 and lib.mgnn_grad_norm_workspace(np_, tp, 3, 0) == -1
  assert lib.mgnn_grad_norm_workspace(None, None, 0, 1) == 0


def test_layer_norm_refusals():
  x = torch.zeros(3, 5, 8)
  w = torch.ones(8)
  for bad, error in (((x.double(),), TypeError), ((x.int(),), TypeError), ((torch.zeros(()),), ValueError), ((torch.zeros(4, 0),), ValueError),
                     ((torch.zeros(1, norm_ops.MAX_COLS + 1),), ValueError), ((x, torch.ones(7)), ValueError), ((x, torch.ones(2, 8)), ValueError),
                     ((x, torch.ones(5, 8)), ValueError), ((x, torch.ones(1, 3, 8)), ValueError), ((x, torch.ones(())), ValueError),
                     ((x, w, torch.ones(3, 8)), ValueError), ((x, w.bfloat16()), TypeError), ((x.half(), w.half(), w), ValueError),
                     ((x.half(), w.bfloat16()), TypeError), ((x, w.to('meta')), ValueError), ((x.to_sparse(),), TypeError)):
    with pytest.raises(error):
      norm_ops.layer_norm(*bad)
  for eps in (-1e-5, float('nan'), float('inf')):
    with pytest.raises(ValueError):
      norm_ops.layer_norm(x, eps=eps)


@pytest.mark.parametrize('dtype', list(norm_ops.TYPES))
def test_layer_norm_on_the_cpu_is_the_formula(dtype):
  g = torch.Generator().manual_seed(1)
  x, w, b = torch.randn(3, 4, 9, generator=g).to(dtype), torch.randn(3, 9, generator=g), torch.randn(3, 9, generator=g)
  y = norm_ops.layer_norm(x, w, b, eps=1e-3)
  xd = x.double()
  h = (xd - xd.mean(-1, keepdim=True)) / torch.sqrt(xd.var(-1, correction=0, keepdim=True) + 1e-3)
  want = h * w.double().unsqueeze(1) + b.double().unsqueeze(1)
  assert y.dtype == dtype and torch.allclose(y.double(), want, rtol=torch.finfo(dtype).eps, atol=1e-5)
  assert torch.equal(norm_ops.layer_norm(x, w[0], None), norm_ops.layer_norm(x, w[0], torch.zeros(9)))
  assert norm_ops.layer_norm(x[:, :0], w, b).shape == (3, 0, 9)
  xg = x.clone().requires_grad_(True)
  norm_ops.layer_norm(xg, w, b).sum().backward()
  assert xg.grad.shape == x.shape


def test_gradient_refusals():
  a, b = torch.ones(3, 4), torch.ones(3)
  for grads, stacked, error in (([a.double()], 0, TypeError), ([a.int()], 0, TypeError), ([a.to_sparse()], 0, TypeError),
                                ([a, torch.ones(3, device='meta')], 0, ValueError), ([a, torch.ones(2)], 3, ValueError),
                                ([torch.ones(())], 1, ValueError), ([a], -1, ValueError), ([a], 1.5, TypeError), ([a, None], 0, TypeError),
                                ([a], norm_ops.MAX_GROUPS + 1, ValueError)):
    with pytest.raises(error):
      norm_ops.grad_norm(grads, stacked)
    with pytest.raises(error):
      norm_ops.clip_grads(grads, 1.0, stacked)
  for max_norm in (-1.0, float('nan')):
    with pytest.raises(ValueError):
      norm_ops.clip_grads([a], max_norm)
  for out in ([], [torch.ones(4, 3)], [a.half()], [a, b], [torch.ones(1, 4).expand(3, 4)]):
    with pytest.raises(ValueError):
      norm_ops.clip_grads([a], 1.0, out=out)


def test_clipping_on_the_cpu_is_the_formula_and_torch_s():
  g = torch.Generator().manual_seed(2)
  params = [torch.nn.Parameter(torch.zeros(s)) for s in ((3, 5, 2), (3,), (3, 7))]
  for p in params:
    p.grad = torch.randn(p.shape, generator=g)
  params.append(torch.nn.Parameter(torch.zeros(3)))      # without a gradient
  grads = [p.grad.clone() for p in params[:3]]
  ref = [torch.nn.Parameter(torch.zeros_like(q)) for q in grads]
  for r, q in zip(ref, grads):
    r.grad = q.clone()
  want = torch.nn.utils.clip_grad_norm_(ref, 0.5)
  out, norm = norm_ops.clip_grads(grads, 0.5)
  assert norm.shape == () and torch.allclose(norm, want) and torch.equal(norm, norm_ops.grad_norm(grads))
  got = norm_ops.clip_grad_norm_(iter(params), 0.5)
  assert torch.equal(got, norm)
  for p, r, o in zip(params, ref, out):
    assert torch.allclose(p.grad, r.grad, rtol=1e-6) and torch.equal(p.grad, o)
  norms = norm_ops.clip_grad_norm_([torch.nn.Parameter(q) for q in grads], 0.5, stacked=3)      # none has a .grad
  assert torch.equal(norms, torch.zeros(3)) and torch.equal(norm_ops.grad_norm([]), torch.zeros(()))
  out, norms = norm_ops.clip_grads(grads, 0.5, stacked=3)
  for a in range(3):
    alone, norm = norm_ops.clip_grads([q[a] for q in grads], 0.5)
    assert torch.allclose(norms[a], norm) and all(torch.allclose(o[a], x) for o, x in zip(out, alone))


def test_layer_norm_policies_on_the_cpu():
  """StackedAgentNets(layer_norm=True) against the stand-alone AgentNets, and their weight files."""
  torch.manual_seed(3)
  st = ppo.StackedAgentNets(2, layer_norm=True)
  with torch.no_grad():
    st.norm1_w.normal_(1, 0.2), st.norm1_b.normal_(0, 0.2), st.norm2_b.normal_(0, 0.2)
  img = torch.randint(0, 11, (2, 17, 5, 5, 3), dtype=torch.uint8)
  d = torch.randint(0, 4, (2, 17))
  logits, values = st(img, d)
  for a in range(2):
    l, v = st.agent_net(a)(img[a], d[a])
    assert torch.allclose(logits[a], l, atol=1e-5) and torch.allclose(values[a], v, atol=1e-5)
  (logits.sum() * 3.0 + values.pow(2).sum()).backward()
  norms = [torch.sqrt(sum(p.grad[a].double().square().sum() for p in st.parameters())) for a in range(2)]
  got = st.clip_grad_norm_(0.5)
  assert torch.allclose(got.double(), torch.stack(norms), rtol=1e-5)
  after = torch.sqrt(sum(p.grad[1].double().square().sum() for p in st.parameters()))
  assert abs(float(after) - min(0.5, float(norms[1]))) < 1e-5
  plain = ppo.StackedAgentNets(2)
  assert len(list(plain.parameters())) == 13
  for to, sd in ((plain, st.agent_state_dict(0)), (st, plain.agent_state_dict(0))):
    with pytest.raises(ValueError):
      to.load_agent_state_dict(0, sd)
  assert set(ppo.AgentNet().state_dict()) == {n for n, _, _ in ppo._STACK}


def test_layer_norm_is_refused_for_the_other_policy():
  class FakeEnv:
    n_agents, n_envs = 2, 4
    obs_image = torch.zeros((2, 4, 5, 5, 3), dtype=torch.uint8)
  with pytest.raises(ValueError):
    ppo.BatchedController(FakeEnv(), ddp=False, policy='multigrid_net', layer_norm=True)
  assert len(list(ppo.BatchedController(FakeEnv(), ddp=False, layer_norm=True).policy.parameters())) == 17
