"""Calls of multigrid_amd/norm_ops.py on the GPU that must be refused, or that must return what simpler calls return."""
import array
import ctypes as C

import pytest
import torch

import norm_abi
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


@pytest.mark.parametrize('value', [1000.0, 4096.0, 30000.0, 1e10, 3.14159e-3, -77777.0])
def test_rows_of_one_value_are_all_zero(value):
  """Every deviation is 0, whatever the mean's rounding; and without eps 0 / 0."""
  for cols in (1, 3, 7, 41, 60, 249, 255, 257, 1000, 1537, 2049, 5000, 9001, 16381):
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
      x = torch.full((3, cols), value, device='cuda').to(dtype)
      if not torch.isfinite(x).all():
        continue
      bias = torch.full((cols,), 2.0, device='cuda')
      xg, wg = x.clone().requires_grad_(True), torch.full((cols,), 3.0, device='cuda', requires_grad=True)
      y = norm_ops.layer_norm(xg, wg, bias)
      assert torch.equal(y, torch.full_like(y, 2.0)), (cols, dtype, float(y[0, 0].detach()))
      dw, = torch.autograd.grad(y, wg, torch.ones_like(y))
      assert not dw.any(), (cols, dtype, float(dw[0]))
      assert torch.isnan(norm_ops.layer_norm(x, eps=0.0)).all(), (cols, dtype)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('mean', [0.0, 300.0, -20000.0])
def test_rows_off_centre_keep_their_deviations(mean, dtype):
  """Deviations of 1 around a mean.  fp32: elements less a first mean m1, off by 40 u of 20000 at most, are exact; their own mean, below 0.9, is
  off by 40 additions, 40 u; the sum of squares by 40 u relative, half of that in the root; x - m1 - shift, its product with
  the root and the root itself by 4 u more.  Together 40 u + 24 u |h|, taken as 44 u (1 + |h|).  16 bits: the mean is rounded to fp32 besides,
  and the result to its type."""
  for cols in (5, 41, 128, 255, 513, 1537, 4100, 9001, 16381):
    x = normal((23, cols), cols, mean, 1.0, dtype)
    xd = x.double()
    m = xd.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((xd - m) ** 2).mean(-1, keepdim=True) + 1e-5)
    want = (xd - m) * rstd
    bound = 44 * U * (1 + want.abs())
    if dtype != torch.float32:
      bound += U * m.abs() * rstd
      bound += (want.abs() + bound) * (torch.finfo(dtype).eps / 2) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    over = (norm_ops.layer_norm(x).double() - want).abs() - bound
    assert float(over.max()) <= 0, (cols, float(over.max()))


def test_saved_tensors_may_come_back_in_another_layout():
  """Hooks on saved tensors (torch.autograd.graph.save_on_cpu) give back a contiguous copy of strided rows; other types, sizes or
  devices are refused."""
  wide = normal((50, 301), 1)
  w, b, dy = normal((130,), 2), normal((130,), 3), normal((50, 130), 4)
  for x in (wide[:, 7:137], wide[::2, 1:131].repeat(2, 1), normal((130, 50), 5).t()):
    def grads(x, w, b):
      xg, wg, bg = (t.detach().requires_grad_(True) for t in (x, w, b))
      return norm_ops.layer_norm(xg, wg, bg), (xg, wg, bg)
    y, leaves = grads(x, w, b)
    want = torch.autograd.grad(y, leaves, dy)
    with torch.autograd.graph.save_on_cpu():
      y, leaves = grads(x, w, b)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, leaves, dy), want))
    # rows that come back further apart than they left
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: torch.cat([t, t], dim=-1)[..., :t.size(-1)]):
      y, leaves = grads(x, w, b)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, leaves, dy), want))
    for unpack in (lambda t: t.cpu(), lambda t: t.half(), lambda t: t[:1]):
      with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        y, leaves = grads(x, w, b)
      with pytest.raises(RuntimeError, match='saved'):
        torch.autograd.grad(y, leaves, dy)


def test_an_older_error_of_the_thread_is_not_this_call_s():
  """hipSetDevice of a device that is not there leaves an error behind; the calls after it succeed and say so."""
  hip = C.CDLL('libamdhip64.so')
  lib = norm_abi.load()
  x, y, norm = normal((6, 20), 1), torch.zeros(6, 20, device='cuda'), torch.zeros(1, device='cuda')
  n, t = array.array('q', [120]), array.array('i', [0])
  src = array.array('Q', [x.data_ptr()])
  stream = torch.cuda.current_stream().cuda_stream
  torch.cuda.synchronize()
  assert hip.hipSetDevice(12345) != 0
  codes = [lib.mgnn_layer_norm(x.data_ptr(), 20, None, None, y.data_ptr(), None, 1, 6, 20, 1e-5, 0, 0, stream)]
  assert hip.hipSetDevice(12345) != 0
  codes.append(lib.mgnn_grad_norm(src.buffer_info()[0], n.buffer_info()[0], t.buffer_info()[0], 1, 1, norm.data_ptr(), None, 0, stream))
  hip.hipGetLastError()
  torch.cuda.synchronize()
  assert codes == [0, 0]
  assert torch.equal(y, norm_ops.layer_norm(x)) and torch.equal(norm[0], norm_ops.grad_norm([x]))


def _leaves(x, w, b):
  return tuple(t.detach().requires_grad_(True) for t in (x, w, b))


SUMS = [(3, 409603, 128, torch.float32), (1, 300007, 64, torch.bfloat16), (2, 100003, 40, torch.bfloat16), (1, 958697, 35, torch.float32),
        (1, 40001, 1024, torch.float16), (2, 5003, 2048, torch.bfloat16), (1, 5003, 1537, torch.float16), (5, 77, 8192, torch.float32),
        (1, 2051, 16384, torch.float32), (1, 1031, 16381, torch.float32), (1, 509, 16384, torch.bfloat16), (70, 1001, 7, torch.float16)]


@pytest.mark.parametrize('agents,rows,cols,dtype', SUMS)
def test_sums_over_rows_count_every_row_once(agents, rows, cols, dtype):
  """Whole numbers, whose sums below 2^24 fp32 holds exactly in any order: dy is odd everywhere, so that every row that is
  missed or counted twice shows.  Rows of a power of 2 of +-1 have mean 0 and variance 1, so that without eps h is x itself."""
  gen = torch.Generator(device='cuda').manual_seed(rows)
  whole = cols & (cols - 1) == 0
  dy = torch.randint(0, 4, (agents, rows, cols), device='cuda', generator=gen, dtype=torch.int8) * 2 - 3
  x = torch.randint(0, 2, (agents, rows, cols // 2), device='cuda', generator=gen, dtype=torch.int8) * 2 - 1
  x = torch.cat([x, -x] + [torch.zeros_like(x[..., :1])] * (cols % 2), dim=-1)
  leaves = _leaves(x.to(dtype), normal((agents, cols), 1), normal((agents, cols), 2))
  y = norm_ops.layer_norm(*leaves, eps=0.0)
  _, dw, db = torch.autograd.grad(y, leaves, dy.to(dtype))
  assert torch.equal(db.long(), dy.sum(-2, dtype=torch.int64)) and torch.equal(db, db.round())
  if whole:
    assert torch.equal(dw.long(), (dy * x).sum(-2, dtype=torch.int64)) and torch.equal(dw, dw.round())


@pytest.mark.parametrize('agents,rows,cols,dtype', SUMS)
def test_a_few_rows_of_many_carry_the_gradient(agents, rows, cols, dtype):
  """dy is 0 but in 24 rows, the first and the last ones among them: sums of 24 terms, to which zeros add nothing.  A sum's terms
  are off by h's error and its own by 24 roundings.  h = (x - m) s: m off by 40 u of the mean |x|, s by 24 u, two operations."""
  x, w, b = normal((agents, rows, cols), 1, 0.4, 1.7, dtype), normal((agents, cols), 2), normal((agents, cols), 3)
  at = torch.cat([torch.arange(8), torch.arange(8) * (rows // 9) + rows // 9 + 1, torch.arange(rows - 8, rows)]).unique().cuda()
  few = normal((agents, len(at), cols), 4, 0, 1, dtype)
  dy = torch.zeros(agents, rows, cols, dtype=dtype, device='cuda')
  dy[:, at] = few
  leaves = _leaves(x, w, b)
  dx, dw, db = torch.autograd.grad(norm_ops.layer_norm(*leaves), leaves, dy)
  xd, d = x[:, at].double(), few.double()
  m = xd.mean(-1, keepdim=True)
  s = 1 / torch.sqrt(((xd - m) ** 2).mean(-1, keepdim=True) + 1e-5)
  h = (xd - m) * s
  dh = 40 * U * xd.abs().mean(-1, keepdim=True) * s + 26 * U * h.abs()
  terms = d * h
  assert ((dw.double() - terms.sum(-2)).abs() <= ((24 * U) * terms.abs() + d.abs() * dh).sum(-2) * 1.01).all()
  assert ((db.double() - d.sum(-2)).abs() <= 24 * U * d.abs().sum(-2) * 1.01).all()
  dx[:, at] = 0
  assert not dx.any()


@pytest.mark.parametrize('agents,rows,cols,dtype,deep', [(3, 409603, 128, torch.float32, 302), (1, 100003, 40, torch.bfloat16, 4)])
def test_sums_over_many_rows_of_real_numbers(agents, rows, cols, dtype, deep):
  """deep: the rows one after the other in a thread, (rows / 8 to a step) over 170 workgroups and (rows / 32) over 782; then at most 3 steps
  over lanes, 2 over waves, 25 and 5 over the workgroups' shares, each a rounding of the sum so far."""
  x, dy = normal((agents, rows, cols), 1, 0.2, 1.0, dtype), normal((agents, rows, cols), 2, 0.1, 1, dtype)
  leaves = _leaves(x, normal((agents, cols), 3, 1.0, 0.2), normal((agents, cols), 4))
  _, dw, db = torch.autograd.grad(norm_ops.layer_norm(*leaves), leaves, dy)
  for a in range(agents):
    xd, d = x[a].double(), dy[a].double()
    m = xd.mean(-1, keepdim=True)
    s = 1 / torch.sqrt(((xd - m) ** 2).mean(-1, keepdim=True) + 1e-5)
    h = (xd - m) * s
    dh = 40 * U * xd.abs().mean(-1, keepdim=True) * s + 26 * U * h.abs()
    terms, steps = d * h, (deep + 36) * U
    assert ((dw[a].double() - terms.sum(-2)).abs() <= (steps * terms.abs() + d.abs() * dh).sum(-2)).all()
    assert ((db[a].double() - d.sum(-2)).abs() <= steps * d.abs().sum(-2)).all()
