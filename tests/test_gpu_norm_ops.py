"""Layer norm with its gradients and clipping by the global gradient norm (include/mgrid_norm.h, multigrid_amd/norm_ops.py)
on the GPU against the formulas in 64 bits.

Tolerances count roundings: u = 2^-24 is half a step of fp32, half a step of an output's type is finfo(type).eps / 2
relative.  A row's mean adds at most 16 elements per thread, 6 lane steps and 16 waves, with a division: its error is
below 40 u times the row's mean |x|; the sum of squared deviations likewise 40 u relative, its root half of that."""
import pytest
import torch

import norm_abi
from multigrid_amd import norm_ops, ppo

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
SMALLEST = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -24}      # one step next to zero


def half_step(want, dtype):
  return want.abs() * (torch.finfo(dtype).eps / 2) + SMALLEST[dtype] / 2


def formula(x, w, b, dy, eps):
  """(y, dx, dw, db) in 64 bits, and the bounds of what the kernels may be off; w, b: [groups, 1, cols]; x: [groups, rows, cols]."""
  x, w, b, dy = (t.double() for t in (x, w, b, dy))
  m = x.mean(-1, keepdim=True)
  v = ((x - m) ** 2).mean(-1, keepdim=True)
  s = 1 / torch.sqrt(v + eps)
  h = (x - m) * s
  y = h * w + b
  e = dy * w
  c1, c2 = e.mean(-1, keepdim=True), (e * h).mean(-1, keepdim=True)
  dx = s * (e - c1 - h * c2)
  dw, db = (dy * h).sum(-2), dy.sum(-2)
  # h is off by the mean's error times s, and by 32 u relative (40 / 2 of s, its own division and root, two operations);
  # a mean that is off by k sigma also adds k^2 to v
  off = 40 * U * x.abs().mean(-1, keepdim=True) * s
  dh = off + (32 * U + off * off) * h.abs()
  ty = dh * w.abs() + 2 * U * (y.abs() + (h * w).abs())
  # the two means over the row are off by 40 u of their terms, and c2 by h's error too
  t1 = 40 * U * e.abs().mean(-1, keepdim=True)
  t2 = 44 * U * (e * h).abs().mean(-1, keepdim=True) + (e.abs() * dh).mean(-1, keepdim=True)
  terms = e.abs() + c1.abs() + (h * c2).abs()
  tx = s * (t1 + h.abs() * t2 + dh * c2.abs() + (32 * U + off * off) * terms)
  # sums over rows: at most 64 rows in a row per thread in these tests, 22 more steps over lanes, waves and workgroups
  tw = 90 * U * (dy * h).abs().sum(-2) + (dy.abs() * dh).sum(-2)
  tb = 90 * U * dy.abs().sum(-2)
  return (y, dx, dw, db), (ty, tx, tw, tb)


def compare(got, want, bound, dtypes, names=('y', 'dx', 'dw', 'db')):
  for g, w, t, d, n in zip(got, want, bound, dtypes, names):
    assert g.dtype == d and g.shape == w.shape, n
    assert torch.isfinite(g).all(), n
    over = (g.double() - w).abs() - t - half_step(w.abs() + t, d)
    assert not over.numel() or float(over.max()) <= 0, (n, float(over.max()), float(t.max()))


def normal(shape, seed, mean=0.0, std=1.0, dtype=F32):
  g = torch.Generator(device='cuda').manual_seed(seed)
  return torch.empty(shape, device='cuda').normal_(mean, std, generator=g).to(dtype)


def both(x, w, b, dy, eps=1e-5):
  xg, wg, bg = (t.detach().requires_grad_(True) for t in (x, w, b))
  y = norm_ops.layer_norm(xg, wg, bg, eps)
  return (y.detach(),) + torch.autograd.grad(y, (xg, wg, bg), dy)


COLS = (1, 2, 3, 7, 8, 9, 16, 31, 33, 64, 65, 100, 128, 255, 257, 512, 513, 1000, 1024, 1025, 1537, 2048, 2049, 4096, 4100, 5000, 8192,
        8193, 12289, 16381, 16384)


@pytest.mark.parametrize('dtype,wdtype', [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
@pytest.mark.parametrize('cols', COLS)
def test_layer_norm_and_gradients(cols, dtype, wdtype):
  for rows in (1, 2, 37, max(1, 60000 // cols)):
    x, dy = normal((1, rows, cols), cols, 0.4, 1.7, dtype), normal((1, rows, cols), cols + 1, 0, 1, dtype)
    w, b = normal((1, cols), cols + 2, 1.0, 0.3, wdtype), normal((1, cols), cols + 3, 0, 0.3, wdtype)
    want, bound = formula(x, w.unsqueeze(1), b.unsqueeze(1), dy, 1e-5)
    y, dx, dw, db = both(x[0], w[0], b[0], dy[0])
    compare((y, dx, dw, db), (want[0][0], want[1][0], want[2][0], want[3][0]), [t[0] for t in bound], (dtype, dtype, wdtype, wdtype))
    assert torch.equal(norm_ops.layer_norm(x[0], w[0], b[0]), y)      # without gradients: the same bits


@pytest.mark.parametrize('agents,rows,cols', [(3, 1, 128), (3, 4096, 64), (3, 1000, 128), (2, 513, 72), (5, 7, 1537), (1, 3, 5), (300, 2, 33), (4, 65, 2000)])
@pytest.mark.parametrize('dtype', [F32, BF16])
def test_stacked_layer_norm(agents, rows, cols, dtype):
  x, dy = normal((agents, rows, cols), 1, -0.3, 2.0, dtype), normal((agents, rows, cols), 2, 0, 1, dtype)
  w, b = normal((agents, cols), 3, 1.0, 0.3), normal((agents, cols), 4, 0, 0.3)
  want, bound = formula(x, w.unsqueeze(1), b.unsqueeze(1), dy, 1e-5)
  compare(both(x, w, b, dy), want, bound, (dtype, dtype, F32, F32))
  # any number of middle axes, and an agent's part alone gives the same bits
  y = norm_ops.layer_norm(x, w, b)
  assert torch.equal(norm_ops.layer_norm(x.reshape(agents, rows, 1, cols), w, b).reshape(x.shape), y)
  assert torch.equal(norm_ops.layer_norm(x[agents - 1], w[agents - 1], b[agents - 1]), y[agents - 1])


@pytest.mark.parametrize('rows', [100003, 3])
def test_many_rows(rows):
  """Sums over many rows: a thread adds at most 1024 rows here before the fixed tree, the bound follows."""
  x, dy = normal((1, rows, 40), 1, 0.2, 1.0, BF16), normal((1, rows, 40), 2, 0.1, 1, BF16)
  w, b = normal((1, 40), 3, 1.0, 0.2), normal((1, 40), 4)
  want, bound = formula(x, w.unsqueeze(1), b.unsqueeze(1), dy, 1e-5)
  bound = (bound[0], bound[1], bound[2] * (1050 / 90), bound[3] * (1050 / 90))
  y, dx, dw, db = both(x[0], w[0], b[0], dy[0])
  compare((y, dx, dw, db), [t[0] for t in want], [t[0] for t in bound], (BF16, BF16, F32, F32))


def test_rows_far_off_centre_and_rows_of_one_value():
  """A mean of 1000 deviations; all elements equal: h is 0 up to the mean's rounding, and eps alone divides."""
  x = normal((1, 65, 515), 1, 1000.0, 1.0)
  w, b, dy = normal((1, 515), 2, 1.0, 0.2), normal((1, 515), 3), normal((1, 65, 515), 4)
  want, bound = formula(x, w.unsqueeze(1), b.unsqueeze(1), dy, 1e-5)
  compare(both(x[0], w[0], b[0], dy[0]), [t[0] for t in want], [t[0] for t in bound], (F32,) * 4)
  for cols in (1, 8, 130, 5000):      # 0.5: every partial sum is exact
    y = norm_ops.layer_norm(torch.full((4, cols), 0.5, device='cuda'), None, torch.full((cols,), 2.0, device='cuda'))
    assert torch.equal(y, torch.full((4, cols), 2.0, device='cuda'))
  zero = norm_ops.layer_norm(torch.zeros(2, 6, device='cuda'), eps=0.0)      # 0 / 0, as the formula says
  assert torch.isnan(zero).all()


def test_tiny_deviations_without_eps():
  """eps = 0 and deviations of 1e-18, whose squares are ordinary fp32 numbers; and of 1e-20, whose squares (1e-40) come in
  steps of 2^-149: off by 7e-6 each, half of that in the root, below 1e-4 with all roundings."""
  for scale, off in ((1e-18, 0.0), (1e-20, 1e-4)):
    x = normal((1, 7, 300), 1) * scale
    w, b, dy = torch.ones(1, 300, device='cuda'), torch.zeros(1, 300, device='cuda'), normal((1, 7, 300), 2)
    want, bound = formula(x, w.unsqueeze(1), b.unsqueeze(1), dy, 0.0)
    got = both(x[0], w[0], b[0], dy[0], 0.0)
    for g, r, t in zip(got, want, bound):
      assert ((g.double() - r[0]).abs() <= t[0] + half_step(r[0].abs() + t[0], F32) + off * r[0].abs().max()).all()


def test_the_largest_number_of_agents():
  n = norm_ops.MAX_GROUPS
  x, w, b, dy = normal((n, 2, 5), 1), normal((n, 5), 2, 1, 0.2), normal((n, 5), 3), normal((n, 2, 5), 4)
  want, bound = formula(x, w.unsqueeze(1), b.unsqueeze(1), dy, 1e-5)
  compare(both(x, w, b, dy), want, bound, (F32,) * 4)
  with pytest.raises(ValueError):
    norm_ops.layer_norm(torch.zeros(n + 1, 2, device='cuda'), torch.zeros(n + 1, 2, device='cuda'))
  check_clip([normal((n, 3), 5), normal((n,), 6)], 0.5, stacked=n)
  check_clip([normal((n, 3), i) for i in range(113)], 0.5, stacked=n)


def test_nan_and_infinity_stay_in_their_row():
  x = normal((6, 777), 1)
  x[1, 5], x[3, 776], x[4, 0] = float('nan'), float('inf'), float('-inf')
  clean = [0, 2, 5]
  w, b, dy = normal((777,), 2), normal((777,), 3), normal((6, 777), 4)
  y, dx, dw, db = both(x, w, b, dy)
  for row in (1, 3, 4):
    assert torch.isnan(y[row]).all() and torch.isnan(dx[row]).all()
  y2, dx2, _, _ = both(x[clean], w, b, dy[clean])
  assert torch.equal(y[clean], y2) and torch.equal(dx[clean], dx2)
  assert torch.isnan(dw).all() and torch.isfinite(db).all()


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_layouts_of_the_input(dtype):
  """Rows in the middle of wider ones, transposed and expanded inputs and gradients, an odd first element."""
  wide = normal((50, 301), 1, 0, 1, dtype)
  w, b = normal((130,), 2, 1.0, 0.2, dtype), normal((130,), 3, 0, 1, dtype)
  flat = normal((50 * 130 + 1,), 4, 0, 1, dtype)
  views = (wide[:, 7:137], wide[::2, 1:131], flat[1:].view(50, 130), normal((130, 50), 5, 0, 1, dtype).t(), wide[:1, :130].expand(50, 130),
           normal((5, 10, 130), 6, 0, 1, dtype).transpose(0, 1), wide[:, :1].expand(50, 130), wide[0, 2:132])
  for x in views:
    dy = normal(x.shape, 7, 0, 1, dtype)
    got, want = both(x, w, b, dy), both(x.contiguous(), w, b, dy)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    for other in (dy[..., :1].expand(x.shape), dy.transpose(0, -1).contiguous().transpose(0, -1)):
      assert all(torch.equal(p, q) for p, q in zip(both(x, w, b, other), both(x.contiguous(), w, b, other.contiguous())))
  every = torch.stack([w, w * 3]).t()      # a weight with stride 2
  assert torch.equal(norm_ops.layer_norm(views[0], every[:, 0], b), norm_ops.layer_norm(views[0], w, b))


def test_nothing_behind_the_rows_is_written():
  """Outputs through the C ABI into the middle of a larger buffer of a known value: its other elements keep it."""
  lib = norm_abi.load()
  stream = torch.cuda.current_stream().cuda_stream
  for dtype, cols, rows in ((F32, 13, 5), (BF16, 37, 70), (F16, 2051, 3), (F32, 16381, 2), (F16, 1, 9)):
    t, n = norm_ops.TYPES[dtype], rows * cols
    x, dy = normal((rows, cols), 1, 0, 1, dtype), normal((rows, cols), 2, 0, 1, dtype)
    room = [torch.full((n + 64,), 7.0, dtype=dtype, device='cuda') for _ in range(2)]
    sums = [torch.full((cols + 64,), 7.0, dtype=dtype, device='cuda') for _ in range(2)]
    stats = torch.full((2 * rows + 64,), 7.0, device='cuda')
    at = [r[31:].data_ptr() for r in room + sums]
    assert lib.mgnn_layer_norm(x.data_ptr(), cols, None, None, at[0], stats.data_ptr(), 1, rows, cols, 1e-5, t, t, stream) == 0
    size = lib.mgnn_layer_norm_workspace(1, rows, cols, t)
    work = torch.full((size // 4 + 64,), 7.0, device='cuda')
    assert lib.mgnn_layer_norm_backward(x.data_ptr(), cols, dy.data_ptr(), None, stats.data_ptr(), at[1], at[2], at[3], work.data_ptr(), size,
                                        1, rows, cols, t, t, stream) == 0
    for r, k in ((room[0], n), (room[1], n), (sums[0], cols), (sums[1], cols)):
      assert (r[:31] == 7).all() and (r[31 + k:] == 7).all(), (dtype, cols)
    assert (stats[2 * rows:] == 7).all() and (work[size // 4:] == 7).all()
    want = both(x, torch.ones(cols, dtype=dtype, device='cuda'), torch.zeros(cols, dtype=dtype, device='cuda'), dy)
    assert torch.equal(room[0][31:31 + n], want[0].flatten()) and torch.equal(room[1][31:31 + n], want[1].flatten())
    assert torch.equal(sums[0][31:31 + cols], want[2]) and torch.equal(sums[1][31:31 + cols], want[3])


def test_parts_of_the_gradient_alone():
  x, w, b, dy = normal((300, 200), 1), normal((200,), 2), normal((200,), 3), normal((300, 200), 4)
  y, dx, dw, db = both(x, w, b, dy)
  for wants in ((True, False, False), (False, True, False), (False, False, True), (False, True, True)):
    leaves = [t.clone().requires_grad_(k) for t, k in zip((x, w, b), wants)]
    got = torch.autograd.grad(norm_ops.layer_norm(*leaves), [t for t in leaves if t.requires_grad], dy)
    assert all(torch.equal(p, q) for p, q in zip(got, [t for t, k in zip((dx, dw, db), wants) if k]))
  xg = x.clone().requires_grad_(True)
  ones, zeros = torch.ones_like(w), torch.zeros_like(b)
  assert torch.equal(torch.autograd.grad(norm_ops.layer_norm(xg), xg, dy)[0], both(x, ones, zeros, dy)[1])
  bg = b.clone().requires_grad_(True)      # a bias alone
  assert torch.equal(torch.autograd.grad(norm_ops.layer_norm(x, None, bg), bg, dy)[0], db)
  with pytest.raises(RuntimeError):        # differentiable once
    first, = torch.autograd.grad(norm_ops.layer_norm(xg, w, b), xg, dy.requires_grad_(True), create_graph=True)
    first.sum().backward()


def test_no_rows():
  w, b = normal((4, 9), 1), normal((4, 9), 2)
  for shape in ((4, 0, 9), (4, 5, 0, 9)):
    x = torch.zeros(shape, device='cuda', requires_grad=True)
    wg, bg = w.clone().requires_grad_(True), b.clone().requires_grad_(True)
    y = norm_ops.layer_norm(x, wg, bg)
    dx, dw, db = torch.autograd.grad(y, (x, wg, bg), torch.zeros_like(y))
    assert y.shape == shape and dx.shape == shape and not dw.any() and not db.any()
  none = norm_ops.layer_norm(torch.zeros(0, 3, 9, device='cuda'), torch.zeros(0, 9, device='cuda'))
  assert none.shape == (0, 3, 9)


def test_gradients_against_differences():
  """Along a random direction: the kernels' gradients against central differences of the formula in 64 bits.  The
  difference quotient is off by h^2 / 6 of a third derivative of order 10, the gradient by fp32 roundings: 2e-5 relative."""
  x, w, b, dy = normal((2, 9, 50), 1), normal((2, 50), 2, 1.0, 0.3), normal((2, 50), 3), normal((2, 9, 50), 4)
  grads = both(x, w, b, dy)[1:]

  def value(x, w, b):
    m = x.mean(-1, keepdim=True)
    h = (x - m) / torch.sqrt(((x - m) ** 2).mean(-1, keepdim=True) + 1e-5)
    return ((h * w.unsqueeze(1) + b.unsqueeze(1)) * dy.double()).sum()
  at = [t.double() for t in (x, w, b)]
  for k in range(3):
    way = normal(at[k].shape, 10 + k).double()
    ends = [[t + s * 1e-4 * way if i == k else t for i, t in enumerate(at)] for s in (1, -1)]
    slope = (value(*ends[0]) - value(*ends[1])) / 2e-4
    got = (grads[k].double() * way).sum()
    assert abs(float(got - slope)) <= 2e-5 * float((grads[k].double().abs() * way.abs()).sum()), k


def test_layer_norm_is_the_same_every_run_and_on_another_stream():
  x, w, b, dy = normal((3, 5000, 130), 1), normal((3, 130), 2), normal((3, 130), 3), normal((3, 5000, 130), 4)
  first = both(x, w, b, dy)
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    second = both(x, w, b, dy)
  torch.cuda.current_stream().wait_stream(side)
  third = both(x, w, b, dy)
  assert all(torch.equal(p, q) and torch.equal(p, r) for p, q, r in zip(first, second, third))


# ---- clipping ----

SIZES = (0, 1, 2, 3, 5, 7, 8, 255, 1023, 4095, 4096, 4097, 8191, 8193, 20000, 100003)


def check_clip(grads, max_norm, stacked=0, flat_out=None):
  """Norms within a rounding to fp32 of a sum in fp64 (whose own 2^-53 steps vanish beside it), results within the factor's
  two roundings and the product's."""
  groups = stacked or 1
  raw = [g.clone() for g in grads]
  sq = sum((g.double().reshape(groups, -1) ** 2).sum(1) for g in raw)
  norm = sq.sqrt()
  out, norms = norm_ops.clip_grads(grads, max_norm, stacked, out=flat_out)
  assert norms.shape == ((stacked,) if stacked else ()) and norms.dtype == F32
  assert ((norms.double().reshape(groups) - norm).abs() <= norm * U * 1.01).all()
  factor = (max_norm / (norm + 1e-6)).clamp(max=1.0)
  for g, r, o in zip(grads, raw, out):
    assert torch.equal(g, r) or any(o is g for o in out)
    want = r.double() * factor.reshape((groups,) + (1,) * (r.dim() - 1) if stacked else ())
    bound = want.abs() * (3 * U) + half_step(want, r.dtype) * 1.01
    assert o.dtype == r.dtype and o.shape == r.shape and ((o.double() - want).abs() <= bound).all()
  assert torch.equal(norm_ops.grad_norm(raw, stacked), norms)
  inplace = [r.clone() for r in raw]
  params = [torch.nn.Parameter(torch.empty_like(r)) for r in inplace]
  for p, r in zip(params, inplace):
    p.grad = r
  assert torch.equal(norm_ops.clip_grad_norm_(params, max_norm, stacked), norms)
  assert all(torch.equal(p.grad, o) for p, o in zip(params, out))
  return out, norms


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('max_norm', [0.5, 1e9, 0.0])
def test_clip_one_tensor_of_every_size(dtype, max_norm):
  for n in SIZES:
    check_clip([normal((n,), n, 0, 0.1, dtype)], max_norm)
    check_clip([normal((2, n), n, 0, 0.1, dtype)], max_norm, stacked=2)


@pytest.mark.parametrize('stacked', [0, 1, 3])
@pytest.mark.parametrize('count', [2, 13, 111, 112, 113, 250])
def test_clip_lists_of_every_length_and_mixed_types(stacked, count):
  kinds = (F32, BF16, F16)
  lead = (stacked,) if stacked else ()
  grads = [normal(lead + (SIZES[i * 7 % len(SIZES)],), i, 0, 0.03 * (1 + i % 3), kinds[i % 3]) for i in range(count)]
  check_clip(grads, 1.0, stacked)


def test_clip_a_list_over_all_launch_shapes():
  """From one workgroup per agent to more chunks than workgroups."""
  for n in (30000, 70000, 200000, 3000001, 20000003):
    check_clip([normal((n,), 1, 0, 0.01), normal((3,), 2)], 0.5)
    check_clip([normal((2, n // 2), 3, 0, 0.01, BF16), normal((2, 1), 4)], 0.5, stacked=2)


def test_clip_a_list_of_many_large_tensors():
  """Ten launches of full grids, whose partial sums are joined by a kernel of their own; norm alone, apart and in place."""
  check_clip([normal((76000 + i,), i, 0, 0.001) for i in range(1120)], 0.5)
  check_clip([normal((2, 76000 + i), i, 0, 0.001, BF16) for i in range(1120)], 0.5, stacked=2)


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_clip_views_of_one_buffer(dtype):
  """Gradients and results as neighbouring parts of flat buffers, none of them aligned."""
  sizes = [1, 7, 100, 33, 4097, 2, 50001]
  flat = normal((sum(sizes) + 1,), 1, 0, 0.05, dtype)
  room = torch.full((sum(sizes) + 6,), 7.0, dtype=dtype, device='cuda')
  cut = lambda t, at: [t[at + sum(sizes[:i]):at + sum(sizes[:i + 1])] for i in range(len(sizes))]      # noqa: E731
  check_clip(cut(flat, 1), 0.5, flat_out=cut(room, 3))
  assert (room[:3] == 7).all() and (room[-3:] == 7).all()
  keep = flat[0].clone()
  norm_ops.clip_grads(cut(flat, 1), 0.5, out=cut(flat, 1))      # in place through views
  assert torch.equal(flat[1:], room[3:-3]) and torch.equal(flat[0], keep)


def test_clip_other_layouts():
  conv = normal((64, 32, 3, 3), 1).contiguous(memory_format=torch.channels_last)
  wide, turned = normal((40, 90), 2), normal((33, 65), 3).t()
  grads = [conv, wide[:, 5:70], turned, normal((5,), 4)[None, :].expand(7, 5)]
  plain, norm = norm_ops.clip_grads([g.contiguous() for g in grads], 0.5)
  out, norm2 = norm_ops.clip_grads(grads, 0.5)
  assert torch.allclose(norm, norm2, rtol=2 * U) and torch.equal(norm_ops.grad_norm(grads), norm2)
  assert all(torch.allclose(p, q, rtol=4 * U, atol=0) for p, q in zip(plain, out))
  edge = wide[:, :5].clone()
  norm_ops.clip_grads(grads[:3], 0.5, out=grads[:3])
  again, _ = norm_ops.clip_grads([torch.ones(2, device='cuda')] * 2, 0.5)      # the same input twice, results apart
  assert torch.equal(again[0], again[1]) and torch.equal(wide[:, :5], edge)
  stacked = normal((7, 3, 5), 5).transpose(0, 1)      # the agent axis is not the outermost in memory
  a, n1 = norm_ops.clip_grads([stacked], 0.5, stacked=3)
  b, n2 = norm_ops.clip_grads([stacked.contiguous()], 0.5, stacked=3)
  assert torch.equal(a[0], b[0]) and torch.equal(n1, n2)
  with pytest.raises(ValueError):
    norm_ops.clip_grads([wide, wide], 0.5, out=[wide, wide])
  with pytest.raises(ValueError):
    norm_ops.clip_grads([wide[:20], wide[19:]], 0.5, out=[wide[:20], wide[19:]])
  with pytest.raises(ValueError):
    norm_ops.clip_grads([wide, torch.ones(3)], 0.5)      # two devices


def test_clip_sees_values_whose_squares_leave_fp32():
  for scale in (1e30, 1e-30):
    g = normal((5000,), 1) * scale
    out, norm = norm_ops.clip_grads([g], scale)
    want = g.double().norm()
    assert abs(float(norm) / float(want) - 1) < 2 * U
    # 1e-6 is part of the factor's formula: at 1e-30 the factor is 1e-24 and the results, of order 1e-54, lie below fp32's
    # smallest number 2^-149, where a rounding is off by up to half of that
    assert torch.allclose(out[0].double(), g.double() * min(1.0, scale / (float(want) + 1e-6)), rtol=4 * U, atol=SMALLEST[F32] / 2)


def test_clip_nan_and_infinity():
  g = [normal((100,), 1), normal((5000,), 2)]
  g[1][4000] = float('inf')
  out, norm = norm_ops.clip_grads(g, 0.5)
  assert torch.isinf(norm) and not out[0].any() and torch.isnan(out[1][4000]) and not out[1][:4000].any()      # inf * 0
  g[0][3] = float('nan')
  out, norm = norm_ops.clip_grads(g, 0.5)
  assert torch.isnan(norm) and all(torch.isnan(o).all() for o in out)
  two = normal((2, 300), 3)
  two[0, 7] = float('nan')
  out, norms = norm_ops.clip_grads([two], 0.5, stacked=2)
  alone, n = norm_ops.clip_grads([two[1:]], 0.5, stacked=1)
  assert torch.isnan(out[0][0]).all() and torch.equal(out[0][1:], alone[0]) and torch.equal(norms[1:], n)
  assert torch.equal(norm_ops.clip_grads([two[1]], float('inf'))[0][0], two[1])


def test_clip_empty_lists_and_tensors():
  empty = torch.zeros(0, device='cuda')
  out, norm = norm_ops.clip_grads([empty, torch.zeros(3, 0, device='cuda')], 0.5)
  assert norm.is_cuda and float(norm) == 0 and out[1].shape == (3, 0)
  out, norms = norm_ops.clip_grads([torch.zeros(3, 0, device='cuda')], 0.5, stacked=3)
  assert torch.equal(norms, torch.zeros(3, device='cuda'))
  out, norm = norm_ops.clip_grads([torch.zeros(40, device='cuda')], 0.5)
  assert float(norm) == 0 and not out[0].any()


def test_in_place_clipping_is_seen_by_autograd():
  g = normal((50,), 1)
  x = torch.ones(50, device='cuda', requires_grad=True)
  y = (x * g).sum()      # saves g
  norm_ops.clip_grads([g], 0.1, out=[g])
  with pytest.raises(RuntimeError):
    y.backward()


def test_captured_clipping_of_a_long_list():
  """More tensors than one launch takes, in place: a graph that fills the gradients and clips them, replayed on new values
  with eager clipping in between."""
  sizes = [1 + 37 * i for i in range(130)] + [300000]
  fresh = [normal((n,), i, 0, 0.1) for i, n in enumerate(sizes)]
  grads = [f.clone() for f in fresh]
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    norm_ops.clip_grads(grads, 0.5, out=grads)
  torch.cuda.current_stream().wait_stream(side)
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    for g, f in zip(grads, fresh):
      g.copy_(f)
    norm = norm_ops.clip_grads(grads, 0.5, out=grads)[1]
  for k in range(4):
    for i, f in enumerate(fresh):
      f.copy_(normal(f.shape, 1000 * k + i, 0, 0.1 + k))
    want, want_norm = norm_ops.clip_grads(fresh, 0.5)
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(norm, want_norm) and all(torch.equal(g, w) for g, w in zip(grads, want)), k


def test_two_streams_at_once():
  """The same operators on two streams without waiting for each other: workspaces are the calls' own."""
  big = [normal((400000,), 1, 0, 0.1), normal((70000,), 2, 0, 0.1, BF16)]
  x, w, b, dy = normal((20000, 130), 3), normal((130,), 4), normal((130,), 5), normal((20000, 130), 6)
  want_clip, want_ln = norm_ops.clip_grads(big, 0.5), both(x, w, b, dy)
  streams = [torch.cuda.Stream(), torch.cuda.Stream()]
  torch.cuda.synchronize()
  got = []
  for k in range(10):
    for st in streams:
      with torch.cuda.stream(st):
        got.append((norm_ops.clip_grads(big, 0.5), both(x, w, b, dy)))
  torch.cuda.synchronize()
  for (out, norm), ln in got:
    assert torch.equal(norm, want_clip[1]) and all(torch.equal(p, q) for p, q in zip(out, want_clip[0]))
    assert all(torch.equal(p, q) for p, q in zip(ln, want_ln))


def test_offsets_past_32_bits():
  """Over 2^31 elements, and over 2^32 to the last row of a strided input: the ends of it against calls on the ends alone."""
  rows, cols = 530000, 4096
  wide = torch.empty((rows, 2 * cols), dtype=BF16, device='cuda').normal_(0.2, 1.5, generator=torch.Generator(device='cuda').manual_seed(1))
  x, w, b = wide[:, 5:5 + cols], normal((cols,), 2, 1, 0.2), normal((cols,), 3)
  dy = torch.ones((rows, cols), dtype=BF16, device='cuda')
  y, dx, dw, db = both(x, w, b, dy)
  for part in (slice(0, 3), slice(262143, 262146), slice(rows - 3, rows)):      # the middle one crosses 2^31 elements of the input
    py, pdx, _, _ = both(x[part], w, b, dy[part])
    assert torch.equal(y[part], py) and torch.equal(dx[part], pdx)
  # every partial sum of ones is a whole number below 2^24
  assert torch.equal(db, torch.full_like(db, float(rows))) and torch.isfinite(dw).all()
  del wide, x, dy, y, dx
  n = 2 ** 31 + 77
  g = torch.full((n,), 0.25, dtype=BF16, device='cuda')
  norm = norm_ops.clip_grads([g], 1.0, out=[g])[1]
  want = 0.25 * n ** 0.5
  assert abs(float(norm) / want - 1) < 2 * U
  value = torch.tensor(0.25 / (want + 1e-6)).to(BF16)      # the same on every element; one step of the type at most from here
  assert bool((g == g[0]).all()) and abs(float(g[0]) / float(value) - 1) <= torch.finfo(BF16).eps


# ---- together, as an update uses them ----

def _net(layer_norm=True):
  torch.manual_seed(0)
  return ppo.StackedAgentNets(3, layer_norm=layer_norm)


def test_layer_norm_policies_equal_the_per_agent_nets():
  """StackedAgentNets(layer_norm=True) against stand-alone AgentNets of the same weights (nn.LayerNorm): outputs, every
  gradient, and the clipped gradients agent by agent."""
  st = _net().cuda()
  img = torch.randint(0, 11, (3, 257, 5, 5, 3), dtype=torch.uint8, generator=torch.Generator().manual_seed(1)).cuda()
  d = torch.randint(0, 4, (3, 257), generator=torch.Generator().manual_seed(2)).cuda()
  with torch.no_grad():
    for name in ('norm1_w', 'norm2_w', 'norm1_b', 'norm2_b'):
      p = getattr(st, name)
      p.add_(normal(p.shape, 3, 0, 0.2))
  logits, values = st(img, d)
  (logits.square().sum() * 3 + values.sum()).backward()
  raw = {n: p.grad.clone() for n, p in st.named_parameters()}
  norms = st.clip_grad_norm_(0.5)
  assert norms.shape == (3,)
  for a in range(3):
    net = st.agent_net(a)
    l, v = net(img[a], d[a])
    # two more roundings-deep layers than without a norm; logits of order 1
    assert torch.allclose(logits[a], l, atol=2e-5) and torch.allclose(values[a], v, atol=2e-5)
    (l.square().sum() * 3 + v.sum()).backward()
    ref = dict(net.named_parameters())
    total = torch.sqrt(sum(p.grad.double().square().sum() for p in ref.values()))
    assert abs(float(norms[a]) / float(total) - 1) < 1e-4
    for ref_name, name, _ in st.stack:
      got, want = raw[name][a], ref[ref_name].grad.reshape(raw[name][a].shape)
      assert float((got - want).double().norm()) <= 1e-4 * float(total), (a, ref_name)
      f = min(1.0, 0.5 / (float(norms[a]) + 1e-6))
      assert torch.allclose(getattr(st, name).grad[a], got * f, rtol=1e-6), (a, ref_name)


def _step(params, x, dy):
  """Two normalised layers, forward and backward, and the clipping of all gradients: an update's use of the operators.
  Between them elementwise torch operations only (torch's reductions are not what is tested)."""
  w1, b1, w2, b2 = params
  h = torch.relu(norm_ops.layer_norm(x, w1, b1))
  y = norm_ops.layer_norm(h * 1.5 + x, w2, b2)
  grads = torch.autograd.grad(y, (x,) + params, dy)
  clipped, norms = norm_ops.clip_grads(grads[1:], 0.1, stacked=3)
  return (y.detach(), grads[0], norms) + tuple(clipped)


def test_a_captured_step_replays_as_the_eager_one():
  """Forward, backward and clipping in two HIP graphs, replayed several times on new inputs, with eager work of the same
  operators between the replays and both graphs at once on two streams: every replay equals the eager step."""
  params = tuple(normal((3, 72), k, k % 2, 0.3).requires_grad_(True) for k in (1, 2, 3, 4))
  xs = [normal((3, 2000, 72), 5).requires_grad_(True), normal((3, 33, 72), 6).requires_grad_(True)]
  dys = [normal(x.shape, 7) for x in xs]
  graphs, outs = [], []
  for x, dy in zip(xs, dys):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
      for _ in range(2):
        _step(params, x, dy)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
      outs.append(_step(params, x, dy))
    graphs.append(g)
  streams = [torch.cuda.Stream(), torch.cuda.Stream()]
  for k in range(4):
    for i, x in enumerate(xs):
      x.detach().copy_(normal(x.shape, 100 + 2 * k + i))
    want = [_step(params, x, dy) for x, dy in zip(xs, dys)]
    torch.cuda.synchronize()
    for s, g in zip(streams, graphs):
      with torch.cuda.stream(s):
        g.replay()
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
      assert all(torch.equal(p, q) for p, q in zip(w, o)), k


def test_training_with_layer_norm_runs_and_clips():
  import multigrid_amd
  env = multigrid_amd.make_batched('MultiGrid-Cluttered-Fixed-15x15', 256, seed=1)
  env.reset()
  ctl = ppo.BatchedController(env, ddp=False, seed=2, layer_norm=True)
  before = ctl.policy.norm1_w.detach().clone()
  losses = ctl.update(ctl.rollout(20))
  assert all(x == x for x in losses) and not torch.equal(before, ctl.policy.norm1_w)
  ctl.amp = BF16      # autocast: 16-bit activations under the norms, fp32 weights
  assert all(x == x for x in ctl.update(ctl.rollout(20)))
  env.close()


def test_the_training_command_with_layer_norm(tmp_path, capsys):
  import json
  from multigrid_amd import train
  train.main(['--envs', '256', '--steps', '10', '--iters', '2', '--window', '1', '--layer-norm', '--hang-dump', '0', '--out', str(tmp_path / 'best')])
  lines = [json.loads(l) for l in capsys.readouterr().out.splitlines() if l.startswith('{')]
  assert [l['iter'] for l in lines] == [0, 1] and all(x == x for l in lines for x in l['loss'])
  weights = torch.load(str(tmp_path / 'best_agent_0.pth'), weights_only=True)
  ppo.AgentNet(layer_norm=True).load_state_dict(weights)


def test_per_agent_nets_are_clipped_one_by_one():
  torch.manual_seed(0)
  nets = ppo.PerAgentNets([ppo.MultiGridPPONet(n_agents=2) for _ in range(2)], all_dirs=True).cuda()
  img = torch.randint(0, 11, (2, 33, 5, 5, 3), dtype=torch.uint8).cuda()
  d = torch.randint(0, 4, (2, 33)).cuda()
  logits, values = nets(img, d)
  (logits[0].sum() * 5 + logits[1].sum() * 1e-4 + values.sum() * 1e-4).backward()
  raw = [[p.grad.clone() for p in net.parameters()] for net in nets.nets]
  nets.clip_grad_norm_(0.5)
  for net, before in zip(nets.nets, raw):
    total = float(torch.sqrt(sum(g.double().square().sum() for g in before)))
    f = min(1.0, 0.5 / (total + 1e-6))
    assert all(torch.allclose(p.grad, g * f, rtol=1e-6, atol=0) for p, g in zip(net.parameters(), before))
