"""Operators of the residual recurrent block at the edges of their ranges, on the GPU: relative precision where values
are small or gates are all but shut, in-place forms, what surrounds a view, and every variant a size can select.

Tolerances as in test_block_ops_gpu.py: u = 2^-24, half a step of the stored type, and the named roundings between.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16, FP8 = torch.float32, torch.bfloat16, torch.float8_e4m3fn
HALF = {F32: U, BF16: 2.0 ** -8}


def rnd(*shape, seed=0, scale=1.0, dtype=F32):
  g = torch.Generator().manual_seed(seed)
  return (torch.randn(*shape, generator=g) * scale).to(dtype)


def close(out, want, rel, what):
  """|out - want| <= (rel + half a step of out's type) |want|, elementwise."""
  o, w = out.detach().cpu().double(), want.double()
  lim = (rel + HALF[out.dtype] * (1 + rel)) * w.abs() + 1e-37
  over = (o - w).abs() > lim
  if bool(over.any()) or not bool(torch.isfinite(o).all()):
    i = int((over | ~torch.isfinite(o)).reshape(-1).nonzero()[0])
    raise AssertionError(f'{what}: {int(over.sum())} of {over.numel()} off, first at {i}: {float(o.reshape(-1)[i])} '
                         f'for {float(w.reshape(-1)[i])}')


# ---- scan: relative precision ---------------------------------------------------------------------


@pytest.mark.parametrize('dt', [F32, BF16])
def test_a_decay_that_is_all_but_shut(hip, dt):
  """The decay sigmoid(-v) and what is multiplied with it, to a few u of themselves however far v is out."""
  v = torch.cat([torch.arange(-30, 31, dtype=F32) * 0.5, torch.tensor([17.0, 20.0, 24.0, 40.0, 80.0, -40.0, -80.0])])
  D = v.numel()
  u, c = v[None].to(dt), torch.zeros(1, D, dtype=dt)
  h, hT, h0 = torch.zeros(1, D, device='cuda', dtype=dt), torch.zeros(1, D, device='cuda'), torch.ones(1, D, device='cuda')
  hip.gated_scan_fwd(u.cuda(), c.cuda(), h, 1, h0=h0, hT=hT, shift=-1.0, cand=None)
  x = u.double() - 1.0
  a = torch.sigmoid(-x)
  # the exponent of e^-v is off by (1.5 |v| + 2) u in all (its rounding, the constant's), and sum, reciprocal,
  # product and exponential by 8 u
  rel = (1.5 * x.abs() + 10) * U
  close(hT, a, rel, 'hT')
  close(h, a, rel, 'h')
  du, dc, dh0 = (torch.zeros(1, D, device='cuda', dtype=t) for t in (dt, dt, F32))
  hip.gated_scan_bwd(torch.ones(1, D, device='cuda', dtype=dt), u.cuda(), c.cuda(), h, du, dc, 1, h0=h0, dh0=dh0, shift=-1.0, cand=None)
  close(dh0, a, rel, 'dh0')
  close(du, -a * torch.sigmoid(x), 2 * rel + 4 * U, 'du')
  close(dc, torch.sigmoid(x), rel, 'dc')


@pytest.mark.parametrize('shift', [-96.0, 31.0, 5.3])
@pytest.mark.parametrize('dt', [F32, BF16])
def test_shifts_that_cancel(hip, dt, shift):
  """Gates near their middle and far from it whose operand and shift are both large."""
  v = torch.arange(-24, 25, dtype=F32) / 2
  u = (v - shift)[None].to(dt)
  D = v.numel()
  h, hT = torch.zeros(1, D, device='cuda', dtype=dt), torch.zeros(1, D, device='cuda')
  hip.gated_scan_fwd(u.cuda(), torch.zeros(1, D, device='cuda', dtype=dt), h, 1, h0=torch.ones(1, D, device='cuda'), hT=hT, shift=shift, cand=None)
  x = u.double() + float(torch.tensor(shift))
  # as in test_a_decay_that_is_all_but_shut, the sum's rounding in the exponent; bf16: the rounding of shift's product
  close(hT, torch.sigmoid(-x), (2.5 * x.abs() + 10 + (abs(shift) if dt == BF16 else 0.0)) * U, 'hT')


@pytest.mark.parametrize('gate', [False, True])
@pytest.mark.parametrize('dt', [F32, BF16])
def test_small_candidates(hip, dt, gate):
  """tanh of small and large candidates, to its own size: in h, and in du (no state) or di (with an input gate)."""
  m = torch.cat([2.0 ** -torch.arange(0, 40, dtype=F32), 0.0625 * (1 + torch.tensor([-2.0, -1.0, 0.0, 1.0, 2.0]) / 128),
                 torch.tensor([0.28125, 0.30078125, 0.3125, 2.0, 5.0, 12.0, 50.0])])
  c = torch.cat([m, -m])[None].to(dt)
  D = c.shape[1]
  u, i = torch.full((1, D), 0.5, dtype=dt), torch.full((1, D), 0.25, dtype=dt)
  kw = dict(i=i.cuda()) if gate else {}
  h, hT = torch.zeros(1, D, device='cuda', dtype=dt), torch.zeros(1, D, device='cuda')
  hip.gated_scan_fwd(u.cuda(), c.cuda(), h, 1, hT=hT, shift=0.0, **kw)
  g = torch.sigmoid(i.double() if gate else u.double())
  want = g * torch.tanh(c.double())
  # tanh's exponential form: 1 - 2 r from 1/16 on (bf16), r to 4 u, so 64 u of itself there; (1 - e) / (1 + e) from 0.3 on
  # (fp32) to 9 u; the gate 8 u
  rel = (80 if dt == BF16 else 24) * U
  close(hT, want, rel, 'hT')
  close(h, want, rel, 'h')
  du, dc, di = (torch.zeros(1, D, device='cuda', dtype=dt) for _ in range(3))
  kb = dict(di=di, **kw) if gate else {}
  hip.gated_scan_bwd(torch.ones(1, D, device='cuda', dtype=dt), u.cuda(), c.cuda(), h, du, dc, 1, shift=0.0, **kb)
  close(di if gate else du, torch.tanh(c.double()) * g * (1 - g), rel + 16 * U, 'di' if gate else 'du')


@pytest.mark.parametrize('dt', [F32, BF16])
def test_long_memories(hip, dt):
  """Two thousand steps of nearly shut and nearly open gates: what survives of the initial state, to its own size."""
  T, D = 2000, 8
  v = torch.tensor([-9.0, -8.0, -7.5, -7.0, -6.5, -6.0, -5.5, 14.0])
  u, c = v.expand(T, D).contiguous().to(dt), torch.zeros(T, D, dtype=dt)
  h, hT = torch.zeros(T, D, device='cuda', dtype=dt), torch.zeros(1, D, device='cuda')
  steps = 2000
  u[1:, 7] = -12.0
  hip.gated_scan_fwd(u.cuda(), c.cuda(), h, T, h0=torch.ones(1, D, device='cuda'), hT=hT, shift=0.0, cand=None)
  want = torch.sigmoid(-u.double()).log().sum(0, keepdim=True).exp()
  # a factor is off by u |v| (1 - a) through the exponent of e^-v, which (1 - a) makes less than u, and 3 u through sum,
  # reciprocal and product; as much again for the multiplications
  close(hT, want, steps * 6 * U, 'hT')


@pytest.mark.parametrize('dt', [F32, BF16])
def test_slopes_of_saturated_candidates_and_gates(hip, dt):
  """dc where tanh is all but flat and di where the input gate is all but open or shut: to their own size."""
  m = torch.arange(1, 33, dtype=F32)
  c = torch.cat([m, -m])[None].to(dt)
  D = c.shape[1]
  i = (1.25 * torch.cat([m, -m]))[None].to(dt)
  u = torch.zeros(1, D, dtype=dt)
  one = torch.ones(1, D, device='cuda', dtype=dt)
  du, dc, di = (torch.zeros(1, D, device='cuda', dtype=dt) for _ in range(3))
  hip.gated_scan_bwd(one, u.cuda(), c.cuda(), one, du, dc, 1, i=i.cuda(), di=di, shift=0.0)
  x, g = c.double(), i.double()
  w = torch.sigmoid(g)
  slope = 4 * torch.exp(-2 * x.abs()) / (1 + torch.exp(-2 * x.abs())) ** 2
  # the exponent 2 |c| of e is off by 3 |c| u (its rounding and the constant's), |i|'s by 1.5 |i| u; e, 1 + e and its
  # reciprocal twice, products: 16 u
  close(dc, w * slope, (3 * x.abs() + 1.5 * g.abs() + 24) * U, 'dc')
  close(di, torch.tanh(x) * w * torch.sigmoid(-g), (3 * g.abs() + 32) * U + (80 if dt == BF16 else 24) * U, 'di')
  hip.gated_scan_bwd(one, u.cuda(), c.cuda(), one, du, dc, 1, shift=0.0)
  close(dc, 0.5 * slope, (3 * x.abs() + 24) * U, 'dc without an input gate')


# ---- rows in 8 bits -------------------------------------------------------------------------------


@pytest.mark.parametrize('dt', [F32, BF16])
@pytest.mark.parametrize('C', [5, 64, 1030, 9001])
def test_small_rows_to_e4m3(hip, dt, C):
  """Rows down to the smallest numbers are scaled as any other row is; a row of zeros is zeros with scale 1."""
  sizes = torch.tensor([1.0, 1e-20, 1e-29, 1e-31, 1e-35, 2e-36, 1e-36, 1e-38, 1e-40, 1e-42, 0.0])
  x = rnd(1, C, seed=1).double().clamp(-3, 3)
  x[0, 0] = 3.5
  x = (x * sizes.double()[:, None]).to(dt)
  q, scale = torch.zeros(len(sizes), C, device='cuda', dtype=FP8), torch.zeros(len(sizes), device='cuda')
  hip.quant_rows(x.cuda(), q, scale)
  most = x.double().abs().amax(1)
  want = torch.where(most > 0, most / 448, torch.ones_like(most))
  # half a step of fp32, a subnormal one below the smallest normal number
  assert bool(((scale.cpu().double() - want).abs() <= 2 * U * want + 2.0 ** -150).all())
  got = q.cpu().float().double()
  # in units of the exact scale: half a step of e4m3 (2^-4 of the value, 2^-10 below its smallest normal), and 4 u of 448
  # through the reciprocal's and the products' roundings
  v = x.double() / want[:, None]
  assert bool(((got - v).abs() <= 2.0 ** -4 * v.abs() + 2.0 ** -10 + 4 * U * 448).all())
  assert bool((got.abs().amax(1)[most > 0] == 448).all()) and bool((got[most == 0] == 0).all())


# ---- operands that share memory -------------------------------------------------------------------


def test_shared_memory_is_refused(hip):
  """Another view of an operand that may be the output itself, parts of an operand, and vectors inside a matrix."""
  buf = torch.zeros(64, 64, device='cuda', dtype=BF16)
  big = torch.zeros(64, 64, device='cuda')
  x, w = torch.zeros(16, 16, device='cuda', dtype=BF16), torch.zeros(16, 16, device='cuda', dtype=BF16)
  y, v, g = (torch.zeros(16, 16, device='cuda', dtype=BF16) for _ in range(3))
  one, ones = torch.ones(16, device='cuda'), torch.ones(16, device='cuda')
  flat = buf.reshape(-1)[:256].view(16, 16)                          # rows of 16 next to each other
  a, b = buf[:16, :16], buf[1:17, :16]                               # rows 64 apart, one row further
  state = big.reshape(-1)[:64].view(4, 16)
  calls = [
      lambda: hip.linear_fwd(x, w, flat, res=a),                     # the same address, another stride
      lambda: hip.linear_fwd(x, w, a, res=b),                        # one row further
      lambda: hip.linear_fwd(x, w, a, z=buf[:16, 8:24]),             # half of its columns
      lambda: hip.linear_fwd(x, w, big[:16, :16], bias=big[3, 4:20]),
      lambda: hip.linear_fwd(flat, w, a),
      lambda: hip.linear_bwd(a, x, w, act='silu', z=v, dz=b),
      lambda: hip.linear_bwd(a, x, w, act='silu', z=b, dz=b[:, :16], dx=buf[2:18, :16]),
      lambda: hip.linear_bwd(x, x, w, dw=g, act='silu', z=v, dz=x),  # dw reads x behind dz
      lambda: hip.linear_bwd(y, x, w, dx=a, dw=b),
      lambda: hip.linear_bwd(y, x, w, dbias=y[0]),
      lambda: hip.rms_norm_fwd(x, one, y, res=a, s=flat),
      lambda: hip.rms_norm_fwd(x, one, y, res=a, s=b),
      lambda: hip.rms_norm_fwd(a, one, y, s=flat),
      lambda: hip.rms_norm_fwd(x, big[0, :16], y, res=big[:16, :16], s=big[:16, :16]),
      lambda: hip.rms_norm_fwd(x, one, y, rstd=one),
      lambda: hip.rms_norm_bwd(y, x, one, ones, a, dres=b),
      lambda: hip.rms_norm_bwd(y, x, one, ones, v, dgamma=one),
      lambda: hip.quant_rows(buf[:16, :16], buf.view(FP8)[:16, :16], one),
      lambda: hip.gated_scan_fwd(x, w, y, 4, h0=state, hT=big.reshape(-1)[16:80].view(4, 16)),
      lambda: hip.gated_scan_fwd(big[:16, :16], big[16:32, :16], big[32:48, :16], 4, first=big[40:56, 3]),
      lambda: hip.gated_scan_fwd(x, w, a, 4, i=b),
      lambda: hip.gated_scan_bwd(y, x, w, v, a, b, 4),
      lambda: hip.gated_scan_bwd(y, x, w, v, a, g, 4, dhT=state, dh0=big.reshape(-1)[16:80].view(4, 16)),
  ]
  for k, call in enumerate(calls):
    with pytest.raises(AssertionError):
      call()
      pytest.fail(f'call {k} was not refused')
  # side by side, and rows in between: no memory is shared
  hip.linear_fwd(buf[:16, :16], w, buf[:16, 16:32], res=buf[:16, 32:48], z=buf[16:32, :16])
  hip.linear_fwd(buf[0:32:2, :16], w, buf[1:32:2, :16])
  hip.gated_scan_fwd(buf[:16, :16], buf[:16, 16:32], buf[:16, 32:48], 4)


# ---- product: every kernel and plan ---------------------------------------------------------------


class View:
  """A [rows, cols] view inside a larger buffer of `around` on the GPU; `whole` says that nothing around it changed."""

  def __init__(self, rows, cols, dtype, left=1, right=8, value=None, around=7.0):
    self.base = torch.full((rows + 1, left + cols + right), around, device='cuda').to(dtype)
    self.t = self.base[:rows, left:left + cols]
    if value is not None:
      self.t.copy_(value)

  def whole(self, what):
    b, t = self.base, self.t
    left = t.storage_offset() % b.shape[1]
    for part in (b[:, :left], b[:, left + t.shape[1]:], b[t.shape[0]:]):
      assert bool((part.float() == 7.0).all()), f'{what}: written outside the view'


def near(out, want, tol, what):
  """|out - want| <= tol + half a step of out's type, elementwise, on the GPU."""
  lim = tol + HALF[out.dtype] * (want.abs() + tol) + 1e-37
  over = ~((out.double() - want).abs() <= lim)
  if bool(over.any()):
    i = over.nonzero()[0]
    raise AssertionError(f'{what}: {int(over.sum())} of {over.numel()} off, first at {i.tolist()}: {float(out[tuple(i)])} '
                         f'for {float(want[tuple(i)])}, allowed {float(lim[tuple(i)])}')


def on_gpu(*shape, seed=0, scale=1.0, dtype=F32):
  g = torch.Generator(device='cuda').manual_seed(seed)
  return (torch.randn(*shape, generator=g, device='cuda') * scale).to(dtype)


def plan_of(hip, what, M, N, K, type=1, act=0, ldr=0, z=0, ldp=None, ldq=None):
  import ctypes
  out = (ctypes.c_int * 8)()
  k, q = ((K, K), (N, K), (N, K))[what]
  assert hip.lib.dd_linear_plan(what, type, M, N, K, ldp or k, ldq or q, act, ldr, z, hip.ws_bytes, out) == 0
  return list(out)


ACTS = {None: 0, 'elu': 1, 'silu': 2, 'gelu': 3}


def slope_and_value(z, act):
  t = z.clone().requires_grad_(True)
  y = {None: lambda: t * 1.0, 'elu': lambda: torch.where(t > 0, t, torch.expm1(t)), 'silu': lambda: t * torch.sigmoid(t),
       'gelu': lambda: t * torch.special.erfc(-t / 2 ** 0.5) / 2}[act]()
  return y.detach(), torch.autograd.grad(y.sum(), t)[0]


# plan: splits above one are written as 2
TILED = [
    (25877, 385, 1041, 'gelu', [1, 256, 256, 1, 0, 0, 0]), (20480, 640, 1040, 'silu', [1, 256, 256, 1, 0, 0, 0]),
    (19845, 515, 1433, None, [1, 256, 256, 1, 0, 0, 0]),
    (16693, 135, 769, 'elu', [1, 192, 128, 1, 0, 0, 0]), (5403, 129, 3915, 'silu', [1, 192, 128, 2, 0, 0, 0]),
    (38727, 397, 1753, 'gelu', [1, 128, 128, 1, 32768, 256, 256]), (27413, 659, 1401, 'silu', [1, 192, 128, 1, 21760, 256, 256]),
    (33129, 403, 1881, 'elu', [1, 128, 128, 2, 32768, 256, 256]), (33313, 131, 1691, 'gelu', [1, 128, 128, 2, 32768, 128, 128]),
    (33519, 269, 1865, 'gelu', [1, 192, 128, 1, 21760, 128, 128]), (35073, 133, 4289, 'silu', [1, 128, 128, 2, 24576, 192, 128]),
]


def few_splits(plan):
  return plan[:3] + [min(plan[3], 2)] + plan[4:7]


@pytest.mark.parametrize('yt', [BF16, F32])
@pytest.mark.parametrize('M,N,K,act,plan', TILED)
def test_tiles_and_launches(hip, M, N, K, act, plan, yt):
  """Ragged products that take each tile shape, split and pair of launches, with all of the epilogue, and the residual
  in place."""
  assert few_splits(plan_of(hip, 0, M, N, K, act=ACTS[act], ldr=N, z=1)) == plan
  x, w = View(M, K, BF16, value=on_gpu(M, K, seed=1)), View(N, K, BF16, value=on_gpu(N, K, seed=2, scale=K ** -0.5))
  b, r = on_gpu(N, seed=3), View(M, N, yt, value=on_gpu(M, N, seed=4))
  y, z = View(M, N, yt), View(M, N, BF16)
  hip.linear_fwd(x.t, w.t, y.t, bias=b, act=act, res=r.t, z=z.t)
  xd, wd = x.t.double(), w.t.double()
  want = xd @ wd.t() + b.double()
  # the instruction adds 16 products to its accumulator at a time: K / 16 + 32 additions, 4 within an instruction
  err = (K / 4 + 48) * U * (xd.abs() @ wd.abs().t()) + 4 * U * want.abs()
  near(z.t, want, err, 'z')
  rd = r.t.double()
  near(y.t, slope_and_value(want, act)[0] + rd, 1.13 * err + 16 * U * (want.abs() + rd.abs()), 'y')
  y.whole('y'), z.whole('z')
  hip.linear_fwd(x.t, w.t, r.t, bias=b, act=act, res=r.t)
  if few_splits(plan_of(hip, 0, M, N, K, act=ACTS[act], ldr=N)) == plan:
    assert torch.equal(r.t, y.t), 'the residual in place'
  else:
    near(r.t, slope_and_value(want, act)[0] + rd, 1.13 * err + 16 * U * (want.abs() + rd.abs()), 'the residual in place')
  r.whole('res')


@pytest.mark.parametrize('M,N,K,act,res,plan', [
    (25445, 385, 855, 'gelu', False, [1, 256, 256, 1, 0, 0, 0]), (25445, 385, 855, None, True, [1, 256, 256, 1, 0, 0, 0]),
    (25445, 385, 2047, 'elu', True, [1, 256, 256, 1, 0, 0, 0]),
    (39339, 389, 1975, 'silu', False, [1, 128, 128, 1, 32768, 256, 256]), (39339, 389, 1975, None, True, [1, 128, 128, 1, 32768, 256, 256]),
    (16693, 135, 1099, 'elu', False, [1, 192, 128, 1, 0, 0, 0]), (16693, 135, 1099, None, True, [1, 192, 128, 1, 0, 0, 0]),
    (28039, 655, 1621, 'gelu', False, [1, 192, 128, 1, 21760, 256, 256]), (28039, 655, 1621, None, True, [1, 192, 128, 1, 21760, 256, 256]),
    (5549, 131, 4873, None, False, [1, 192, 128, 2, 0, 0, 0]), (32803, 429, 2355, None, True, [1, 128, 128, 2, 32768, 256, 256])])
def test_tiles_and_launches_e4m3(hip, M, N, K, act, res, plan):
  assert few_splits(plan_of(hip, 0, M, N, K, type=2, act=ACTS[act], ldr=N if res else 0)) == plan
  x = View(M, K, FP8, value=on_gpu(M, K, seed=1, scale=60.0).clamp(-448, 448).to(FP8))
  w = View(N, K, FP8, value=on_gpu(N, K, seed=2, scale=60.0).clamp(-448, 448).to(FP8))
  sx, sw, b = on_gpu(M, seed=3).abs() * 0.01 + 1e-3, on_gpu(N, seed=4).abs() * 1e-3 + 1e-4, on_gpu(N, seed=5)
  r, y = View(M, N, BF16, value=on_gpu(M, N, seed=6)) if res else None, View(M, N, BF16)
  hip.linear_fwd(x.t, w.t, y.t, bias=b, act=act, res=r.t if res else None, x_scale=sx, w_scale=sw)
  xd, wd = x.t.float().double(), w.t.float().double()
  s = sx.double()[:, None] * sw.double()
  want = (xd @ wd.t()) * s + b.double()
  eights = lambda t: torch.nn.functional.pad(t, (0, -K % 8)).reshape(t.shape[0], -1, 8).abs().amax(2)  # noqa: E731
  # sums as in bf16, and of eight consecutive products what is below 2^-13 of the largest: less than 7 2^-13 of it
  err = ((K / 4 + 48) * U * (xd.abs() @ wd.abs().t()) + 7 * 2.0 ** -13 * (eights(xd) @ eights(wd).t())) * s + 8 * U * want.abs()
  rd = r.t.double() if res else torch.zeros_like(want)
  near(y.t, slope_and_value(want, act)[0] + rd, 1.13 * err + 16 * U * (want.abs() + rd.abs()), 'y')
  y.whole('y')


@pytest.mark.parametrize('M,N,K,what,plan', [
    (2701, 103, 4433, 1, [1, 256, 256, 1, 0, 0, 0]), (605, 8711, 4383, 1, [1, 256, 256, 2, 0, 0, 0]),
    (4135, 529, 4397, 1, [1, 128, 128, 1, 3584, 256, 256]), (5641, 461, 3597, 1, [1, 192, 128, 1, 4352, 256, 256]),
    (2307, 2537, 3569, 1, [1, 128, 128, 2, 2304, 128, 128]),
    (269, 1723, 4777, 2, [1, 256, 256, 1, 0, 0, 0]), (22203, 131, 2295, 2, [1, 256, 256, 2, 0, 0, 0]),
    (521, 3861, 4231, 2, [1, 128, 128, 1, 3840, 256, 256]), (2167, 2691, 2953, 2, [1, 128, 128, 2, 2688, 128, 128])])
def test_tiles_and_launches_of_gradients(hip, M, N, K, what, plan):
  assert few_splits(plan_of(hip, what, M, N, K)) == plan
  x, w = View(M, K, BF16, value=on_gpu(M, K, seed=1)), View(N, K, BF16, value=on_gpu(N, K, seed=2, scale=K ** -0.5))
  dy = View(M, N, BF16, value=on_gpu(M, N, seed=3))
  d = dy.t.double()
  if what == 1:
    dx, wd = View(M, K, BF16), w.t.double()
    hip.linear_bwd(dy.t, x.t, w.t, dx=dx.t)
    near(dx.t, d @ wd, (N / 4 + 48) * U * (d.abs() @ wd.abs()), 'dx')
    dx.whole('dx')
    return
  xd = x.t.double()
  want, err = d.t() @ xd, (M / 4 + 48) * U * (d.abs().t() @ xd.abs())
  old = on_gpu(N, K, seed=4)
  for acc in (False, True):
    dw = View(N, K, F32, value=old)
    hip.linear_bwd(dy.t, x.t, w.t, dw=dw.t, accumulate=acc)
    near(dw.t, want + old.double() if acc else want, err + 2 * U * (want.abs() + old.double().abs()), 'dw')
    dw.whole('dw')


def test_long_rows_of_many_outputs(hip):
  """Sixteen rows at most with long contractions stay with the few-row kernel however many outputs there are."""
  M, N, K = 8, 17001, 4100
  assert plan_of(hip, 0, M, N, K)[:2] == [0, 16]
  x, w = on_gpu(M, K, seed=1, dtype=BF16), on_gpu(N, K, seed=2, scale=K ** -0.5, dtype=BF16)
  y = View(M, N, BF16)
  hip.linear_fwd(x, w, y.t)
  want = x.double() @ w.double().t()
  near(y.t, want, (K / 4 + 48) * U * (x.double().abs() @ w.double().abs().t()), 'y')
  y.whole('y')


@pytest.mark.parametrize('accumulate', [False, True])
def test_general_kernel_split(hip, accumulate):
  """Rows megabytes apart, whose contraction is split over the general kernel's workgroups, in all three products."""
  M, N, K, ld = 5, 1003, 1000, (1 << 21) + 2
  assert plan_of(hip, 0, M, 40, K, ldp=ld)[:2] == [2, 4] and plan_of(hip, 1, M, N, 40, ldp=ld)[:2] == [2, 4]
  far = torch.empty(M, ld, device='cuda', dtype=BF16)
  x, w, dz = far[:, 3:3 + K], on_gpu(N, K, seed=2, dtype=BF16), far[:, 5001:5001 + N]
  x.copy_(on_gpu(M, K, seed=1)), dz.copy_(on_gpu(M, N, seed=3))
  y, b = View(M, 40, F32), on_gpu(40, seed=4)
  hip.linear_fwd(x, w[:40], y.t, bias=b)
  xd, wd = x.double(), w.double()
  near(y.t, xd @ wd[:40].t() + b.double(), (K / 4 + 50) * U * (xd.abs() @ wd[:40].abs().t() + b.double().abs()), 'y')
  dx = View(M, 40, F32)
  hip.linear_bwd(dz, x[:, :40], w[:, :40], dx=dx.t)
  near(dx.t, dz.double() @ wd[:, :40], (N / 4 + 48) * U * (dz.double().abs() @ wd[:, :40].abs()), 'dx')
  y.whole('y'), dx.whole('dx')
  M, N, K, ld = 530, 24, 70, (1 << 23) + 2
  assert plan_of(hip, 2, M, N, K, ldp=ld)[:2] == [2, 2]
  far = torch.empty(M, ld, device='cuda', dtype=BF16)
  dz, x = far[:, 7:7 + N], on_gpu(M, K, seed=5, dtype=BF16)
  dz.copy_(on_gpu(M, N, seed=6))
  old = on_gpu(N, K, seed=7)
  dw = View(N, K, F32, value=old)
  hip.linear_bwd(dz, x, on_gpu(N, K, seed=8, dtype=BF16), dw=dw.t, accumulate=accumulate)
  d, xd = dz.double(), x.double()
  want = d.t() @ xd + (old.double() if accumulate else 0.0)
  near(dw.t, want, (M / 4 + 48) * U * (d.abs().t() @ xd.abs()) + 2 * U * want.abs(), 'dw')
  dw.whole('dw')


# ---- in place -------------------------------------------------------------------------------------


@pytest.mark.parametrize('yt', [BF16, F32])
@pytest.mark.parametrize('M,N,K', [(8, 2048, 1024), (13, 47, 200), (40, 521, 520), (100, 1001, 520), (70, 95, 256), (300, 257, 1030),
                                   (1300, 301, 1031), (700, 1021, 333), (257, 129, 8200), (1000, 200, 2048)])
def test_residual_in_place(hip, M, N, K, yt):
  """y over res, bit for bit what another output gets: few rows, small tiles, tiles, a split contraction; rows whose last
  columns overlap their neighbour's."""
  x, w = on_gpu(M, K, seed=1, dtype=BF16), on_gpu(N, K, seed=2, scale=K ** -0.5, dtype=BF16)
  r, y, b = View(M, N, yt, value=on_gpu(M, N, seed=3)), View(M, N, yt), on_gpu(N, seed=4)
  for act in (None, 'gelu'):
    hip.linear_fwd(x, w, y.t, bias=b, act=act, res=r.t)
    stream = View(M, N, yt, value=r.t)
    hip.linear_fwd(x, w, stream.t, bias=b, act=act, res=stream.t)
    assert torch.equal(stream.t, y.t)
    stream.whole('stream')


@pytest.mark.parametrize('act', ['elu', 'silu', 'gelu'])
@pytest.mark.parametrize('N', [1, 7, 9, 65, 515, 1021])
@pytest.mark.parametrize('M', [3, 256, 300, 5001])
def test_activation_gradient_in_place(hip, M, N, act):
  """dz over dy and over z, with the same dbias, dx and dw as from a tensor of its own."""
  K = 24
  x, w = on_gpu(M, K, seed=1, dtype=BF16), on_gpu(N, K, seed=2, dtype=BF16)
  dy, z = (View(M, N, BF16, value=on_gpu(M, N, seed=k)) for k in (3, 4))
  got = []
  for which in ('apart', 'dy', 'z'):
    d, t = View(M, N, BF16, value=dy.t), View(M, N, BF16, value=z.t)
    dz = {'apart': View(M, N, BF16), 'dy': d, 'z': t}[which]
    db, dx, dw = torch.zeros(N, device='cuda'), torch.zeros(M, K, device='cuda'), torch.zeros(N, K, device='cuda')
    hip.linear_bwd(d.t, x, w, dx=dx, dw=dw, dbias=db, act=act, z=t.t, dz=dz.t)
    for v in (d, t, dz):
      v.whole(which)
    got.append((dz.t, db, dx, dw))
  for other in got[1:]:
    assert all(torch.equal(a, b) for a, b in zip(got[0], other))
  zd = z.t.double()
  near(got[0][0], dy.t.double() * slope_and_value(zd, act)[1], 32 * U * dy.t.double().abs() * (1 + zd.abs()), 'dz')


@pytest.mark.parametrize('C', [1, 7, 9, 33, 100, 1024, 1542, 2051, 4099, 8195, 16389])
@pytest.mark.parametrize('t', [F32, BF16])
def test_sum_over_x(hip, C, t):
  """s over x, with and without a residual."""
  rows = 37
  x, res, g = on_gpu(rows, C, seed=1, dtype=t), on_gpu(rows, C, seed=2, dtype=t), 1 + on_gpu(C, seed=3, scale=0.1)
  for r in (None, res):
    out = []
    for over in (False, True):
      v = View(rows, C, t, value=x)
      s, y, rstd = View(rows, C, t), View(rows, C, BF16), torch.zeros(rows, device='cuda')
      hip.rms_norm_fwd(v.t, g, y.t, rstd=rstd, res=r, s=v.t if over else s.t)
      out.append(((v if over else s).t, y.t, rstd))
      v.whole('x'), s.whole('s'), y.whole('y')
    assert all(torch.equal(a, b) for a, b in zip(*out))
    assert torch.equal(out[0][0], x if r is None else (x.float() + r.float()).to(t))


# ---- norm: more rows than workgroups --------------------------------------------------------------


@pytest.mark.parametrize('over', [False, True])
@pytest.mark.parametrize('rows,C,workgroups,per', [
    (120001, 64, 1536, 32), (50001, 17, 1536, 32), (13001, 300, 1536, 4), (7001, 1000, 768, 4), (4001, 1542, 1536, 1),
    (2001, 2500, 768, 1), (700, 8101, 256, 1), (701, 9001, 256, 1), (600, 20001, 256, 1)])
def test_norm_gradients_of_many_rows(hip, rows, C, workgroups, per, over):
  """More rows than are in flight at once (`per` of a workgroup), no multiple of them: a workgroup goes round its loop two
  or three times."""
  slots = workgroups * per
  assert rows > slots and rows % slots
  for t in (F32, BF16):
    s, dy, dres, g = on_gpu(rows, C, seed=1, dtype=t), on_gpu(rows, C, seed=2, dtype=BF16), on_gpu(rows, C, seed=3, dtype=t), 1 + on_gpu(C, seed=4, scale=0.1)
    rstd = 1 / s.float().square().mean(1).sqrt()
    dr = View(rows, C, t, value=dres)
    ds, dgamma = dr if over else View(rows, C, t), torch.zeros(C, device='cuda')
    hip.rms_norm_bwd(dy, s, rstd, g, ds.t, dgamma, dr.t)
    inv = rstd.double()[:, None]
    n, d = s.double() * inv, dy.double()
    dn = d * g.double()
    size = dres.double().abs() + inv * (dn.abs() + n.abs() * (dn * n).abs().mean(1, keepdim=True))
    # the row's mean: 32 elements of a lane, 6 steps over a wave, 16 waves
    near(ds.t, dres.double() + inv * (dn - n * (dn * n).mean(1, keepdim=True)), 64 * U * size, 'ds')
    # dgamma: the rows of a lane, up to 32 rows of a workgroup, the workgroups in 32 runs and then those; n and a product
    chain = rows / slots + 1 + per + workgroups / 32 + 32 + 4
    near(dgamma, (d * n).sum(0), chain * U * (d * n).abs().sum(0), 'dgamma')
    ds.whole('ds')


# ---- what surrounds a view ------------------------------------------------------------------------


@pytest.mark.parametrize('M,N,K', [(300, 260, 1030), (300, 257, 1031), (1300, 301, 577), (257, 129, 8201), (2500, 515, 1542), (40, 33, 1030),
                                   (70, 61, 77), (19845, 515, 433)])
def test_what_surrounds_a_view_is_not_read_as_data(hip, M, N, K):
  """Rows and columns around every operand hold NaN: the results are those of compact operands, bit for bit."""
  x, w, r = on_gpu(M, K, seed=1, dtype=BF16), on_gpu(N, K, seed=2, scale=K ** -0.5, dtype=BF16), on_gpu(M, N, seed=3, dtype=BF16)
  dy, z, b = on_gpu(M, N, seed=4, dtype=BF16), on_gpu(M, N, seed=5, dtype=BF16), on_gpu(N, seed=6)
  nan = float('nan')
  results = []
  for left in (None, 3, 8):
    put = lambda t: t if left is None else View(*t.shape, t.dtype, left, 5, value=t, around=nan).t  # noqa: E731
    bias = b if left is None else torch.cat([b.new_full((1,), nan), b, b.new_full((1,), nan)])[1:-1]
    y, y32, kept = torch.zeros(M, N, device='cuda', dtype=BF16), torch.zeros(M, N, device='cuda'), torch.zeros(M, N, device='cuda', dtype=BF16)
    hip.linear_fwd(put(x), put(w), y, bias=bias, act='gelu', res=put(r), z=kept)
    hip.linear_fwd(put(x), put(w), y32, res=put(r.float()))
    dx, dw, db, dz = (torch.zeros(*s, device='cuda', dtype=t) for s, t in [((M, K), BF16), ((N, K), F32), ((N,), F32), ((M, N), BF16)])
    hip.linear_bwd(put(dy), put(x), put(w), dx=dx, dw=dw, dbias=db, act='silu', z=put(z), dz=dz if left is None else put(dz))
    results.append((y, y32, kept, dx, dw, db))
  for k, t in enumerate(results[0]):
    assert bool(torch.isfinite(t).all())
    for other in results[1:]:
      assert torch.equal(t, other[k]), k


@pytest.mark.parametrize('M,N,K', [(300, 260, 1030), (1300, 301, 577), (25445, 385, 855), (40, 33, 1030), (70, 61, 77)])
def test_what_surrounds_rows_in_8_bits(hip, M, N, K):
  x, w = (on_gpu(*s, seed=k, scale=60.0).clamp(-448, 448).to(FP8) for k, s in ((1, (M, K)), (2, (N, K))))
  sx, sw = on_gpu(M, seed=3).abs() * 0.01, on_gpu(N, seed=4).abs() * 1e-3
  y, y2 = (torch.zeros(M, N, device='cuda', dtype=BF16) for _ in range(2))
  hip.linear_fwd(x, w, y, x_scale=sx, w_scale=sw)
  hip.linear_fwd(View(M, K, FP8, 3, 5, value=x, around=float('nan')).t, View(N, K, FP8, 3, 5, value=w, around=float('nan')).t, y2, x_scale=sx, w_scale=sw)
  assert bool(torch.isfinite(y).all()) and torch.equal(y, y2)
