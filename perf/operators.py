"""The trainer's normalisation operators, case by case: layer norm with its gradients, and clipping by the global
gradient norm.

`run(state)` computes one case, in its plain form (elementary torch operations in 32 bits) or, with `own = True`, through
multigrid_amd.norm_ops.  `exact(case, seed)` is the same answer in 64 bits.

Layer norm over the last axis of x, for every row: m = mean(x), v = mean((x - m)^2), h = (x - m) / sqrt(v + eps),
y = h * w + b.  With a leading agent axis (agents > 0) x is [agents, rows, cols] and w, b are [agents, cols].
Clipping: n = sqrt(sum of every gradient's squares), every gradient times min(1, max_norm / (n + 1e-6)); with a leading
agent axis on every gradient, each agent has a norm of its own.
"""
import math

import torch

own = False

EPS = 1e-5
DTYPES = {'float32': torch.float32, 'bfloat16': torch.bfloat16, 'float16': torch.float16}


def listed():
  def ln(name, agents, rows, cols, dtype, wdtype, train):
    return {'name': name, 'op': 'layer_norm', 'agents': agents, 'rows': rows, 'cols': cols, 'dtype': dtype,
            'wdtype': wdtype, 'train': train}

  def clip(name, net, agents, depth, width, dtype, vdtype, flat, max_norm):
    return {'name': name, 'op': 'clip_grads', 'net': net, 'agents': agents, 'depth': depth, 'width': width, 'dtype': dtype,
            'vdtype': vdtype, 'flat': flat, 'max_norm': max_norm}
  return [
      # three agents choose one action each in a single env: the first hidden layer of their stacked policies
      ln('ln_one_env', 3, 1, 128, 'float32', 'float32', False),
      # one rollout step of 4096 envs
      ln('ln_rollout_step', 3, 4096, 128, 'float32', 'float32', False),
      # one epoch of an update over 4096 envs x 100 steps, first hidden layer
      ln('ln_update', 3, 409600, 128, 'float32', 'float32', True),
      # the same epoch under autocast, second hidden layer: activations in 16 bits, weights in 32
      ln('ln_update_amp', 3, 409600, 64, 'bfloat16', 'float32', True),
      # a wide network's training batch, everything in bfloat16
      ln('ln_wide', 0, 16384, 4096, 'bfloat16', 'bfloat16', True),
      # a width and a batch that fit no tile
      ln('ln_odd', 0, 5003, 1537, 'float16', 'float16', True),
      # a few very long rows, odd as well
      ln('ln_long_rows', 0, 509, 16381, 'float32', 'float32', True),
      # one agent's policy network, 37,544 gradients in 13 tensors
      clip('clip_one_policy', 'policy', 0, 0, 0, 'float32', 'float32', False, 0.5),
      # the stacked policies of three agents, clipped agent by agent, as an update does it
      clip('clip_stacked', 'policy', 3, 0, 0, 'float32', 'float32', False, 0.5),
      # an odd-sized network, matrices in bfloat16 and vectors in 32 bits, gradients still in the all-reduce's flat buffers
      clip('clip_odd_mixed', 'mlp', 0, 9, 1021, 'bfloat16', 'float32', True, 1.0),
      # a network whose gradient norm stays below the bound, so that the gradients come out as they went in
      clip('clip_not_needed', 'mlp', 0, 8, 4096, 'bfloat16', 'bfloat16', False, 1e6),
      # half a billion gradients in 32 bits
      clip('clip_large', 'mlp', 0, 8, 8192, 'float32', 'float32', False, 1.0),
  ]


def _log_int(rng, low, high):
  return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
  agents = rng.choice((0, 0, 1, 2, 3, 5))
  dtype = rng.choice(tuple(DTYPES))
  if rng.random() < 0.6:
    cols = _log_int(rng, 8, 16384)
    elements = _log_int(rng, 64, 1 << 26)
    return {'op': 'layer_norm', 'agents': agents, 'rows': max(1, elements // (cols * max(1, agents))), 'cols': cols,
            'dtype': dtype, 'wdtype': rng.choice((dtype, 'float32')), 'train': rng.random() < 0.6}
  depth = rng.randint(1, 12)
  return {'op': 'clip_grads', 'net': 'mlp', 'agents': agents, 'depth': depth, 'width': _log_int(rng, 3, 2500), 'dtype': dtype,
          'vdtype': rng.choice((dtype, 'float32')), 'flat': rng.random() < 0.5, 'max_norm': rng.choice((0.5, 1.0, 1.0, 1e6))}


def _shapes(case):
  """[(shape, dtype name)] of a network's gradients, the leading agent axis included."""
  lead = (case['agents'],) if case['agents'] else ()
  if case['net'] == 'policy':     # the policy network of multigrid_amd.ppo: two convolutions, an embedding, four linear layers
    shapes = [(32, 3, 3, 3), (32,), (64, 32, 3, 3), (64,), (4, 8), (128, 72), (128,), (64, 128), (64,), (7, 64), (7,), (1, 64), (1,)]
    return [(lead + s, case['dtype']) for s in shapes]
  w = case['width']               # depth layers: weight, bias, and a layer norm's weight and bias
  layer = [(lead + (w, w), case['dtype'])] + [(lead + (w,), case['vdtype'])] * 3
  return layer * case['depth']


def _views(case, device):
  """Uninitialised tensors of the case's shapes: consecutive views of one buffer per type (flat), or one by one."""
  shapes = _shapes(case)
  if not case['flat']:
    return [torch.empty(s, dtype=DTYPES[d], device=device) for s, d in shapes]
  room = {d: torch.empty(sum(math.prod(s) for s, t in shapes if t == d), dtype=DTYPES[d], device=device) for _, d in shapes}
  used, out = dict.fromkeys(room, 0), []
  for s, d in shapes:
    out.append(room[d][used[d]:used[d] + math.prod(s)].view(s))
    used[d] += math.prod(s)
  return out


def prepare(case, seed):
  dev = torch.device('cuda')
  gen = torch.Generator(device=dev).manual_seed(seed)
  if case['op'] == 'clip_grads':
    grads = _views(case, dev)
    for i, g in enumerate(grads):  # layers' gradients differ in scale; bounds of 0.5 and 1 clip most networks
      g.normal_(0.0, 0.02 * (1 + i % 4), generator=gen)
    return {'case': dict(case), 'grads': grads, 'out': _views(case, dev)}
  shape = ((case['agents'],) if case['agents'] else ()) + (case['rows'], case['cols'])
  wshape = shape[:-2] + shape[-1:]

  def normal(s, mean, std, dtype):
    return torch.empty(s, dtype=DTYPES[dtype], device=dev).normal_(mean, std, generator=gen)
  # pre-activations of a linear layer: off centre; weights and biases around a layer norm's start of 1 and 0
  x = normal(shape, 0.3, 1.5, case['dtype'])
  w, b = normal(wshape, 1.0, 0.2, case['wdtype']), normal(wshape, 0.0, 0.2, case['wdtype'])
  if not case['train']:
    return {'case': dict(case), 'x': x, 'w': w, 'b': b}
  return {'case': dict(case), 'x': x.requires_grad_(), 'w': w.requires_grad_(), 'b': b.requires_grad_(),
          'dy': normal(shape, 0.0, 1.0, case['dtype'])}


def _own(state):
  from multigrid_amd import norm_ops
  case = state['case']
  if case['op'] == 'clip_grads':
    out, norms = norm_ops.clip_grads(state['grads'], case['max_norm'], stacked=case['agents'], out=state['out'])
    return {'grads': out, 'norm': norms}
  x, w, b = state['x'], state['w'], state['b']
  y = norm_ops.layer_norm(x, w, b, eps=EPS)
  if not case['train']:
    return {'y': y}
  dx, dw, db = torch.autograd.grad(y, (x, w, b), state['dy'])
  return {'y': y, 'dx': dx, 'dw': dw, 'db': db}


def _plain_layer_norm(state):
  case, x = state['case'], state['x'].float()
  w, b = state['w'].float(), state['b'].float()
  if case['agents']:
    w, b = w.unsqueeze(1), b.unsqueeze(1)
  d = x - x.mean(dim=-1, keepdim=True)
  rstd = 1.0 / torch.sqrt((d * d).mean(dim=-1, keepdim=True) + EPS)
  h = d * rstd
  y = (h * w + b).to(state['x'].dtype)
  if not case['train']:
    return {'y': y}
  dy = state['dy'].float()
  dh = dy * w
  dx = rstd * (dh - dh.mean(dim=-1, keepdim=True) - h * (dh * h).mean(dim=-1, keepdim=True))
  return {'y': y, 'dx': dx.to(y.dtype), 'dw': (dy * h).sum(dim=-2).to(state['w'].dtype), 'db': dy.sum(dim=-2).to(state['b'].dtype)}


def _plain_clip(state):
  case, grads = state['case'], state['grads']
  groups = max(1, case['agents'])
  norms = torch.stack([g.float().square().reshape(groups, -1).sum(dim=1) for g in grads]).sum(dim=0).sqrt()
  coef = (case['max_norm'] / (norms + 1e-6)).clamp(max=1.0)
  out = [(g.float().reshape(groups, -1) * coef.unsqueeze(1)).reshape(g.shape).to(g.dtype) for g in grads]
  return {'grads': out, 'norm': norms if case['agents'] else norms[0]}


def run(state):
  if own:
    return _own(state)
  with torch.no_grad():
    return _plain_clip(state) if state['case']['op'] == 'clip_grads' else _plain_layer_norm(state)


def exact(case, seed):
  state = prepare(case, seed)
  if case['op'] == 'clip_grads':
    a = case['agents']
    squares = [torch.linalg.vector_norm(g.double().flatten(1 if a else 0), dim=-1) ** 2 for g in state['grads']]
    norm = torch.sqrt(sum(squares))
    scale = torch.minimum(torch.ones_like(norm), case['max_norm'] / (norm + 1e-6))
    return {'grads': [g.double() * scale.reshape(scale.shape + (1,) * (g.dim() - scale.dim())) for g in state['grads']],
            'norm': norm}
  x, w, b = (state[k].detach().double().requires_grad_(case['train']) for k in 'xwb')
  rows_w, rows_b = (w.unsqueeze(-2), b.unsqueeze(-2)) if case['agents'] else (w, b)
  v, m = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
  y = torch.addcmul(rows_b, (x - m) / torch.sqrt(v + EPS), rows_w)
  if not case['train']:
    return {'y': y}
  dx, dw, db = torch.autograd.grad(y, (x, w, b), state['dy'].double())
  return {'y': y.detach(), 'dx': dx, 'dw': dw, 'db': db}


def work(case):
  size = {'float32': 4, 'bfloat16': 2, 'float16': 2}
  if case['op'] == 'clip_grads':
    n = [(math.prod(s), size[d]) for s, d in _shapes(case)]
    return {'bytes': 2 * sum(k * b for k, b in n) + 4 * max(1, case['agents']), 'flops': 3 * sum(k for k, _ in n)}
  lead = max(1, case['agents'])
  n, m = lead * case['rows'] * case['cols'], lead * case['cols']
  if not case['train']:           # reads x, w, b; writes y
    return {'bytes': 2 * n * size[case['dtype']] + 2 * m * size[case['wdtype']], 'flops': 7 * n}
  # reads x, dy, w, b; writes y, dx, dw, db
  return {'bytes': 4 * n * size[case['dtype']] + 4 * m * size[case['wdtype']], 'flops': 19 * n}
