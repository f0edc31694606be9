"""Operators of the residual recurrent block on the GPU against float64 restatements
(oracle/ref_ops.py) on the same inputs.

Tolerances come from the arithmetic.  u = 2^-24 is half a step of fp32; storing a result adds half a
step of its type relative to the value (bf16 2^-8, e4m3 2^-4 above its smallest normal).  A sum of n terms
whose longest chain of additions is d is off by at most d u times the sum of the terms' magnitudes; the
chains are named where they are used.  exp and reciprocal instructions: one ulp, the exponent's scaling
|x| u, together below 16 u for the arguments here.
"""

import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16, FP8 = torch.float32, torch.bfloat16, torch.float8_e4m3fn
HALF = {F32: U, BF16: 2.0 ** -8}


def rnd(*shape, seed=0, scale=1.0, dtype=F32):
  g = torch.Generator().manual_seed(seed)
  return (torch.randn(*shape, generator=g) * scale).to(dtype)


class Slot:
  """A [rows, cols] view inside a larger buffer on the GPU; `whole` says that nothing around it changed."""

  def __init__(self, rows, cols, dtype, left=0, right=0, below=1, value=None):
    ld = left + cols + right
    self.base = torch.full(((rows + below), ld), 7.0, device='cuda').to(dtype)
    self.t = self.base[:rows, left:left + cols]
    if value is not None:
      self.t.copy_(value)
    self.inside = torch.zeros_like(self.base, dtype=torch.bool)
    self.inside[:rows, left:left + cols] = True

  def whole(self):
    assert bool((self.base.float()[~self.inside] == 7.0).all()), 'written outside the view'


def within(out, want, tol, what=''):
  """|out - want| <= tol + half a step of out's type, elementwise; non-finite values in the same places."""
  o, w = out.detach().cpu().double(), want.double()
  fin = torch.isfinite(w)
  assert torch.equal(torch.isfinite(o), fin), f'{what}: non-finite values differ'
  tol = tol if torch.is_tensor(tol) else torch.full_like(w, tol)
  lim = tol + HALF.get(out.dtype, 0.0) * (w.abs() + tol) + 1e-37
  over = ((o - w).abs() > lim) & fin
  if bool(over.any()):
    i = int(over.reshape(-1).nonzero()[0])
    raise AssertionError(f'{what}: {int(over.sum())} of {over.numel()} off, first at {i}: {float(o.reshape(-1)[i])} '
                         f'for {float(w.reshape(-1)[i])}, allowed {float(lim.reshape(-1)[i])}')


# ---- norm -----------------------------------------------------------------------------------------

NORM_SHAPES = [(4, 8), (3, 9), (700, 1542), (2, 515), (3, 1025), (2, 4097), (1, 16390), (1, 1), (3, 7), (8, 64), (5, 1542), (130, 1024), (257, 512), (6, 2050), (2, 8192), (3, 9001), (1, 32768),
               (1000, 64), (3333, 100), (77, 200), (130, 17), (61, 256)]


@pytest.mark.parametrize('rows,C', NORM_SHAPES)
@pytest.mark.parametrize('xt,rt', [(F32, F32), (BF16, F32), (BF16, BF16), (F32, BF16)])
def test_norm(hip, ref, rows, C, xt, rt):
  left = 8 if C % 8 == 0 else 1      # aligned column slices, and rows of any alignment
  x, r, g = rnd(rows, C, seed=1, dtype=xt), rnd(rows, C, seed=2, scale=2.0, dtype=rt), 1 + rnd(C, seed=3, scale=0.1)
  dy, dres = rnd(rows, C, seed=4, dtype=xt), rnd(rows, C, seed=5, dtype=rt)
  xs, rs, ss, ys = (Slot(rows, C, t, left, 8, value=v) for t, v in [(xt, x), (rt, r), (rt, None), (xt, None)])
  rstd = torch.zeros(rows, device='cuda')
  hip.rms_norm_fwd(xs.t, g.cuda(), ys.t, rstd=rstd, res=rs.t, s=ss.t)
  s, y, inv = torch.zeros(rows, C, dtype=rt), torch.zeros(rows, C).double(), torch.zeros(rows).double()
  ref.rms_norm_fwd(x, g, y, rstd=inv, res=r, s=s)
  assert torch.equal(ss.t.cpu(), s)
  # chain of the mean: 32 elements of a lane, 6 steps over a wave, 16 waves; half of it through the root
  within(rstd, inv, 32 * U * inv, 'rstd')
  within(ys.t, y, 40 * U * y.abs(), 'y')
  ds, dd = Slot(rows, C, rt, left, 8), torch.zeros(rows, C).double()
  dys, drs = Slot(rows, C, xt, left, 8, value=dy), Slot(rows, C, rt, left, 8, value=dres)
  dg0 = rnd(C, seed=6)
  dgamma, dgr = dg0.cuda(), dg0.double()
  hip.rms_norm_bwd(dys.t, ss.t, rstd, g.cuda(), ds.t, dgamma, drs.t, accumulate=True)
  ref.rms_norm_bwd(dy, s, inv, g, dd, dgr, dres, accumulate=True)
  n = s.double() * inv[:, None]
  dn = (dy.double() * g.double()).abs()
  size = dres.double().abs() + inv[:, None] * (dn + n.abs() * (dn * n.abs()).mean(1, keepdim=True))
  within(ds.t, dd, 100 * U * size, 'ds')
  # chain of dgamma: the rows of a lane, 4 waves, partial rows of a workgroup in sixteenths
  within(dgamma, dgr, (64 + rows / 64 + 64) * U * (dg0.double().abs() + (dy.double() * n).abs().sum(0)), 'dgamma')
  for t in (xs, rs, ss, ys, ds):
    t.whole()


@pytest.mark.parametrize('rows,C', [(1, 5), (9, 64), (33, 1024), (4, 1542), (2, 12000), (300, 100), (77, 33)])
@pytest.mark.parametrize('norm', [True, False])
def test_rows_to_e4m3(hip, ref, rows, C, norm):
  x, r, g = rnd(rows, C, seed=7, dtype=BF16), rnd(rows, C, seed=8), 1 + rnd(C, seed=9, scale=0.1)
  x[rows // 2] = 0 if not norm else x[rows // 2]
  q, scale = Slot(rows, C, FP8, 0, 16 if C % 8 == 0 else 3), torch.zeros(rows, device='cuda')
  if norm:
    hip.rms_norm_fwd(x.cuda(), g.cuda(), q.t, res=r.cuda(), s=torch.zeros(rows, C, device='cuda'), scale=scale)
    want = torch.zeros(rows, C).double()
    ref.rms_norm_fwd(x, g, want, res=r, s=torch.zeros(rows, C))
  else:
    hip.quant_rows(x.cuda(), q.t, scale)
    want = x.double()
  most = want.abs().amax(1)
  want_scale = torch.where(most > 0, most / 448, torch.ones_like(most))
  within(scale, want_scale, 48 * U * want_scale, 'scale')
  got = q.t.cpu().float().double() * scale.cpu().double()[:, None]
  # half a step of e4m3: 2^-4 of the value, 2^-10 of the scale below the smallest normal value
  tol = 2.0 ** -4 * want.abs() + 2.0 ** -10 * want_scale[:, None] + 100 * U * most[:, None]
  assert bool(((got - want).abs() <= tol).all())
  assert bool((q.t.cpu().float().abs().amax(1)[most > 0] == 448).all()), 'the largest value of a row is 448 steps of its scale'
  q.whole()


def test_norm_in_place_and_without_residual(hip, ref):
  x, r, g = rnd(40, 256, seed=1, dtype=BF16), rnd(40, 256, seed=2), 1 + rnd(256, seed=3, scale=0.1)
  y1, y2, s = (torch.zeros(40, 256, device='cuda') for _ in range(3))
  hip.rms_norm_fwd(x.cuda(), g.cuda(), y1, res=r.cuda(), s=s)
  stream = r.cuda()
  hip.rms_norm_fwd(x.cuda(), g.cuda(), y2, res=stream, s=stream)       # the stream is updated in place
  assert torch.equal(y1, y2) and torch.equal(s, stream)
  y3, want = torch.zeros(40, 256, device='cuda', dtype=BF16), torch.zeros(40, 256).double()
  hip.rms_norm_fwd(x.cuda(), g.cuda(), y3)
  ref.rms_norm_fwd(x, g, want)
  within(y3, want, 40 * U * want.abs(), 'no residual')


def test_norm_rows_do_not_mix(hip):
  """Non-finite and zero rows leave their neighbours alone; a zero row gives zeros."""
  x = rnd(9, 1542, seed=1)
  clean = torch.zeros(9, 1542, device='cuda')
  g = torch.ones(1542, device='cuda')
  hip.rms_norm_fwd(x.cuda(), g, clean)
  x[2, 5], x[4, 1541], x[6] = float('nan'), float('inf'), 0.0
  y = torch.zeros(9, 1542, device='cuda')
  hip.rms_norm_fwd(x.cuda(), g, y)
  keep = [0, 1, 3, 5, 7, 8]
  assert torch.equal(y[keep], clean[keep])
  assert bool(torch.isnan(y[2]).all()) and bool(torch.isnan(y[4, 1541])) and bool((y[6] == 0).all())


@pytest.mark.parametrize('C', [33, 100, 1024, 1542, 4099, 16389])
@pytest.mark.parametrize('rt', [F32, BF16])
def test_norm_in_place_at_any_width(hip, C, rt):
  """s over res and ds over dres give what separate outputs give: no wave of a row reads what another wrote."""
  rows = 37
  x, r, dy, dres = (rnd(rows, C, seed=k, dtype=t).cuda() for k, t in [(1, BF16), (2, rt), (3, BF16), (4, rt)])
  g = (1 + rnd(C, seed=5, scale=0.1)).cuda()
  y, y2, s, ds = (torch.zeros(rows, C, device='cuda', dtype=t) for t in (BF16, BF16, rt, rt))
  rstd, rstd2 = torch.zeros(rows, device='cuda'), torch.zeros(rows, device='cuda')
  hip.rms_norm_fwd(x, g, y, rstd=rstd, res=r, s=s)
  stream = r.clone()
  hip.rms_norm_fwd(x, g, y2, rstd=rstd2, res=stream, s=stream)
  assert torch.equal(stream, s) and torch.equal(y2, y) and torch.equal(rstd2, rstd)
  hip.rms_norm_bwd(dy, s, rstd, g, ds, None, dres)
  hip.rms_norm_bwd(dy, s, rstd, g, dres, None, dres)
  assert torch.equal(dres, ds)


# ---- product --------------------------------------------------------------------------------------

LINEAR_SHAPES = [(1300, 301, 1031), (20, 70, 1031), (50, 40, 4100), (1300, 1030, 520), (2500, 520, 1542), (130, 2048, 1544), (5000, 1024, 72), (257, 129, 8200), (1, 1, 1), (1, 64, 512), (3, 5, 7), (8, 2048, 1024), (17, 130, 40), (33, 96, 1542), (64, 64, 64), (65, 65, 65),
                 (100, 256, 4096), (129, 515, 72), (300, 200, 1030), (257, 1024, 512), (1000, 384, 640)]


def dot_error(x, w, K):
  """Bound of the sum's error: the instruction adds 16 products to its accumulator at a time, over at most
  8 partial sums and 16 slabs; no chain is longer than K / 16 + 32 additions, and 4 within an instruction."""
  return (K / 4 + 48) * U * (x.double().abs() @ w.double().abs().t())


@pytest.mark.parametrize('M,N,K', LINEAR_SHAPES)
@pytest.mark.parametrize('act,yt', [(None, BF16), ('silu', BF16), ('gelu', F32), ('elu', BF16)])
def test_linear(hip, ref, M, N, K, act, yt):
  al = K % 8 == 0 and N % 8 == 0
  x, w = rnd(M, K, seed=1, dtype=BF16), rnd(N, K, seed=2, scale=K ** -0.5, dtype=BF16)
  b, r = rnd(N, seed=3), rnd(M, N, seed=4, dtype=yt)
  left = 8 if al else 1
  xs, ws, rs = Slot(M, K, BF16, left, 8, value=x), Slot(N, K, BF16, 0, 8, value=w), Slot(M, N, yt, left, 8, value=r)
  ys, zs = Slot(M, N, yt, left, 8), Slot(M, N, BF16, left, 8)
  hip.linear_fwd(xs.t, ws.t, ys.t, bias=b.cuda(), act=act, res=rs.t, z=zs.t)
  y, z = torch.zeros(M, N).double(), torch.zeros(M, N).double()
  ref.linear_fwd(x, w, y, bias=b, act=act, res=r, z=z)
  err = dot_error(x, w, K) + 4 * U * z.abs()
  within(zs.t, z, err, 'z')
  # |act'| <= 1.13; the activations are good to 16 u of their argument
  within(ys.t, y, 1.13 * err + 16 * U * (z.abs() + r.double().abs()), 'y')
  ys.whole(), zs.whole()


@pytest.mark.parametrize('M,N,K', LINEAR_SHAPES)
@pytest.mark.parametrize('act,pt', [(None, F32), ('silu', BF16), ('gelu', BF16), ('elu', F32)])
def test_linear_gradients(hip, ref, M, N, K, act, pt):
  al = K % 8 == 0 and N % 8 == 0
  left = 8 if al else 1
  x, w, dy = rnd(M, K, seed=1, dtype=BF16), rnd(N, K, seed=2, scale=K ** -0.5, dtype=BF16), rnd(M, N, seed=3, dtype=BF16)
  z = rnd(M, N, seed=4, scale=2.0, dtype=BF16)
  xs, ws, dys, zs = (Slot(a.shape[0], a.shape[1], BF16, left, 8, value=a) for a in (x, w, dy, z))
  dx, dw, dz = Slot(M, K, BF16, left, 8), Slot(N, K, pt, left, 8), Slot(M, N, BF16, left, 8)
  old = rnd(N, seed=5, dtype=pt)
  db = old.cuda()
  hip.linear_bwd(dys.t, xs.t, ws.t, dx.t, dw.t, None, act=act, z=zs.t, dz=dz.t)
  hip.linear_bwd(dys.t, xs.t, ws.t, dbias=db, act=act, z=zs.t, dz=dz.t, accumulate=True)
  g = dy.double() * ref._act(z.double(), act)[1]
  if act:
    within(dz.t, g, 32 * U * dy.double().abs() * (1 + z.double().abs()), 'dz')
    gq = dz.t.cpu()            # the products read the stored dz
  else:
    gq = dy
  within(dx.t, gq.double() @ w.double(), dot_error(gq, w.t(), N), 'dx')
  within(dw.t, gq.double().t() @ x.double(), dot_error(gq.t(), x.t(), M), 'dw')
  size = (dy.double() * ref._act(z.double(), act)[1]).abs() + 32 * dy.double().abs() * (1 + z.double().abs()) / (M + 64)
  within(db, old.double() + g.sum(0), (M + 64) * U * (size.sum(0) + old.double().abs()), 'dbias')
  for t in (dx, dw):
    t.whole()
  if act:
    dz.whole()
  before = dw.t.clone()
  hip.linear_bwd(dys.t, xs.t, ws.t, dw=dw.t, act=act, z=zs.t, dz=dz.t, accumulate=True)
  within(dw.t, 2 * before.cpu().double(), dot_error(gq.t(), x.t(), M) * 2 + HALF[pt] * 4 * before.cpu().double().abs(), 'accumulate')


def groups_of_eight(x):
  K = x.shape[1]
  return torch.nn.functional.pad(x.double(), (0, -K % 8)).reshape(x.shape[0], -1, 8)


def eight_error(x, w):
  """Bound of what the 8-bit matrix instruction cuts off (test_e4m3_products_are_added_in_eights): of each of eight
  consecutive products less than u = 2^(E - 13), E the largest sum of their operands' exponents.  The product with
  that sum has magnitude 2^E at least and loses nothing (its last place is 2^(E - 6)), so the other seven lose less than
  7 2^-13 times the largest product, which is at most the product of the largest operands."""
  return 7 * 2.0 ** -13 * groups_of_eight(x).abs().amax(2) @ groups_of_eight(w).abs().amax(2).t()


@pytest.mark.parametrize('rows', [16, 64, 256])
def test_e4m3_products_are_added_in_eights(hip, rows):
  """The instruction's arithmetic bit for bit, in every kernel that uses it: eight consecutive products, each cut towards zero
  to a multiple of 2^(E - 13), E the largest of the eight sums of operand exponents; their sum is exact."""
  x, w = (rnd(rows, 8, seed=k, scale=60.0).clamp(-448, 448).to(FP8).float() for k in (1, 2))
  long = torch.zeros(rows, 600)
  long[:, 592:] = w                                  # (600: past the general kernel's short contractions)
  cases = [(x, w), (torch.nn.functional.pad(x, (592, 0)), long)]
  xe, we = (torch.floor(torch.log2(t.double().abs().clamp(min=2.0 ** -9))) for t in (x, w))
  prod = x.double()[:, None] * w.double()[None]
  unit = 2.0 ** ((xe[:, None] + we[None]).amax(2, keepdim=True) - 13)
  want = (torch.trunc(prod / unit) * unit).sum(2)
  one = torch.ones(rows, device='cuda')
  for a, b in cases:
    y = torch.zeros(rows, rows, device='cuda')
    hip.linear_fwd(a.to(FP8).cuda(), b.to(FP8).cuda(), y, x_scale=one, w_scale=one)
    assert torch.equal(y.cpu().double(), want)


@pytest.mark.parametrize('M,N,K', [(1, 16, 16), (5, 7, 9), (32, 1024, 4096), (16, 48, 128), (65, 130, 200), (300, 257, 1030), (700, 512, 256), (2100, 1040, 1030), (3000, 1000, 528), (700, 300, 4111), (20, 33, 515)])
@pytest.mark.parametrize('act', [None, 'gelu'])
def test_linear_e4m3(hip, ref, M, N, K, act):
  x, w = rnd(M, K, seed=1, scale=60.0).clamp(-448, 448).to(FP8), rnd(N, K, seed=2, scale=60.0).clamp(-448, 448).to(FP8)
  sx, sw, b = rnd(M, seed=3).abs() * 0.01 + 1e-3, rnd(N, seed=4).abs() * 1e-3 + 1e-4, rnd(N, seed=5)
  r = rnd(M, N, seed=6, dtype=BF16)
  xs, ws, ys = Slot(M, K, FP8, 0, 16 if K % 16 == 0 else 3, value=x), Slot(N, K, FP8, 0, 16 if K % 16 == 0 else 3, value=w), Slot(M, N, BF16, 8, 8)
  hip.linear_fwd(xs.t, ws.t, ys.t, bias=b.cuda(), act=act, res=r.cuda(), x_scale=sx.cuda(), w_scale=sw.cuda())
  y, z = torch.zeros(M, N).double(), torch.zeros(M, N).double()
  ref.linear_fwd(x.float(), w.float(), y, bias=b, act=act, res=r, z=z, x_scale=sx, w_scale=sw)
  err = (dot_error(x.float(), w.float(), K) + eight_error(x.float(), w.float())) * sx.double()[:, None] * sw.double() + 8 * U * z.abs()
  within(ys.t, y, 1.13 * err + 16 * U * (z.abs() + r.double().abs()), 'y')
  ys.whole()


def test_linear_residual_in_place_and_rows_do_not_mix(hip):
  x, w, r = rnd(70, 256, seed=1, dtype=BF16).cuda(), rnd(96, 256, seed=2, dtype=BF16).cuda(), rnd(70, 96, seed=3, dtype=BF16).cuda()
  y = torch.zeros(70, 96, device='cuda', dtype=BF16)
  hip.linear_fwd(x, w, y, res=r)
  stream = r.clone()
  hip.linear_fwd(x, w, stream, res=stream)
  assert torch.equal(y, stream)
  x[3, 100], x[40, 255] = float('nan'), float('inf')
  y2 = torch.zeros_like(y)
  hip.linear_fwd(x, w, y2, res=r)
  keep = [i for i in range(70) if i not in (3, 40)]
  assert torch.equal(y2[keep], y[keep]) and bool(torch.isnan(y2[3]).all()) and not bool(torch.isfinite(y2[40]).any())


@pytest.mark.parametrize('act,yt', [('gelu', BF16), ('silu', F32)])
@pytest.mark.parametrize('M,N,K', [(3001, 1541, 453), (10001, 2049, 517), (33001, 260, 1542)])
def test_linear_many_tiles(hip, ref, M, N, K, act, yt):
  """Products of more than one round of tiles, whose last rows may run in another launch and tile shape."""
  test_linear(hip, ref, M, N, K, act, yt)


@pytest.mark.parametrize('M,N,K', [(3001, 453, 1541), (517, 7751, 2050)])
def test_linear_gradients_many_tiles(hip, ref, M, N, K):
  test_linear_gradients(hip, ref, M, N, K, 'silu', F32)


@pytest.mark.parametrize('act,yt', [(None, F32), ('gelu', BF16)])
@pytest.mark.parametrize('M,N,K', [(65, 700, 1000), (97, 333, 1031), (128, 520, 4104), (111, 2391, 577), (7, 16401, 300), (40, 8301, 520),
                                   (100, 4201, 520), (33, 20001, 24)])
def test_linear_a_hundred_rows(hip, ref, M, N, K, act, yt):
  test_linear(hip, ref, M, N, K, act, yt)
  test_linear_e4m3(hip, ref, M, N, K, act)


@pytest.mark.parametrize('M,N,K', [(3001, 1541, 903), (2500, 2048, 1536), (16501, 1030, 1040)])
def test_linear_e4m3_many_tiles(hip, ref, M, N, K):
  test_linear_e4m3(hip, ref, M, N, K, 'silu')


@pytest.mark.parametrize('M', [3, 70, 300])
@pytest.mark.parametrize('act', ['elu', 'silu', 'gelu'])
def test_activations_at_extremes(hip, ref, M, act):
  """Arguments from the smallest to the largest, and NaN, in every variant of the epilogue (few rows, tiles, and
  a contraction of one element)."""
  N = 24
  z = torch.tensor([0.0, 1e-30, -1e-30, 0.25, -0.25, -0.3125, 5.0, -5.0, 20.0, -20.0, 88.0, -88.0, 1e4, -1e4, 3e38, -3e38]).to(BF16)
  w = torch.cat([z, z[:8]])[:, None].cuda()
  x = torch.ones(M, 1, device='cuda', dtype=BF16)
  y = torch.zeros(M, N, device='cuda')
  hip.linear_fwd(x, w, y, act=act)
  zz = w.cpu().double().t().expand(M, N)
  want = ref._act(zz, act)[0]
  within(y, want, 16 * U * zz.abs(), act)
  x[1] = float('nan')
  hip.linear_fwd(x, w, y, act=act)
  assert bool(torch.isnan(y[1]).all()) and bool(torch.isfinite(y[0]).all()) and bool(torch.isfinite(y[2]).all())


@pytest.mark.parametrize('ld', [(1 << 20) - 6, (1 << 23) + 2])
def test_linear_rows_far_apart(hip, ld):
  """Operands and outputs whose rows are megabytes apart (offsets past 2^31 elements and 2^32 bytes), in the tiled
  and in the general kernel: the results of compact ones."""
  M, N, K = (5000 if ld < 1 << 22 else 300), 40, 64
  far = [torch.empty(M, ld, device='cuda', dtype=BF16) for _ in range(2)]
  assert far[0].numel() > 1 << 31
  x, w, r = rnd(M, K, seed=1, dtype=BF16), rnd(N, K, seed=2, dtype=BF16), rnd(M, N, seed=3, dtype=BF16)
  xs, ys, zs, rs = far[0][:, 5:5 + K], far[1][:, 3:3 + N], far[1][:, 100:100 + N], far[0][:, 200:200 + N]
  xs.copy_(x), rs.copy_(r)
  hip.linear_fwd(xs, w.cuda(), ys, res=rs, z=zs)
  want = x.double() @ w.double().t()
  err = dot_error(x, w, K)
  within(zs, want, err, 'z')
  within(ys, want + r.double(), err + 2 * U * (want.abs() + r.double().abs()), 'y')
  dx, dw = far[1][:, 300:300 + K], torch.zeros(N, K, device='cuda')
  hip.linear_bwd(rs, xs, w.cuda(), dx=dx, dw=dw)
  within(dx, r.double() @ w.double(), dot_error(r, w.t(), N), 'dx')
  within(dw, r.double().t() @ x.double(), dot_error(r.t(), x.t(), M), 'dw')


def test_linear_ragged_columns_hold_anything(hip):
  """Columns behind K in the rows of x and w are not read as data: NaN there changes nothing."""
  for K in (40, 72, 1030):
    xs, ws = torch.full((50, 1040), float('nan'), device='cuda', dtype=BF16), torch.full((64, 1040), float('nan'), device='cuda', dtype=BF16)
    x, w = rnd(50, K, seed=1, dtype=BF16).cuda(), rnd(64, K, seed=2, dtype=BF16).cuda()
    xs[:, :K], ws[:, :K] = x, w
    y, y2 = (torch.zeros(50, 64, device='cuda') for _ in range(2))
    hip.linear_fwd(x, w, y)
    hip.linear_fwd(xs[:, :K], ws[:, :K], y2)
    assert bool(torch.isfinite(y2).all())
    assert float((y - y2).abs().max()) <= 2 * (K / 4 + 48) * U * float((x.float().abs() @ w.float().abs().t()).max())


# ---- scan -----------------------------------------------------------------------------------------


def restarts(B, T, p, seed):
  g = torch.Generator().manual_seed(seed)
  f = (torch.rand(B, T, generator=g) < p).float()
  return f.reshape(-1)


def linear_recurrence(a, b, x):
  out = []
  for t in range(a.shape[1]):
    x = a[:, t] * x + b[:, t]
    out.append(x)
  return torch.stack(out, 1)


SCAN_SHAPES = [(1, 1, 1), (3, 1, 64), (64, 1, 1024), (2, 3, 7), (1, 8, 130), (5, 9, 33), (2, 50, 256), (3, 33, 515), (2, 127, 64),
               (1, 128, 64), (1, 300, 192), (2, 1000, 96), (1, 4097, 64), (300, 40, 70)]


@pytest.mark.parametrize('B,T,D', SCAN_SHAPES)
@pytest.mark.parametrize('gate,cand,dt', [(False, 'tanh', F32), (True, None, F32), (False, None, BF16), (True, 'tanh', BF16)])
def test_scan(hip, ref, B, T, D, gate, cand, dt):
  n = 3 if gate else 2
  parts = Slot(B * T, n * D, dt, 0, 8 if D % 8 == 0 else 1, value=rnd(B * T, n * D, seed=1, scale=1.5, dtype=dt))
  cols = [parts.t[:, k * D:(k + 1) * D] for k in range(n)] + [None]
  u, c, i = cols[0], cols[1], cols[2] if gate else None
  host = [None if t is None else t.cpu() for t in (u, c, i)]
  first = restarts(B, T, 0.04, 2) if T > 1 else torch.tensor([1.0] + [0.0] * (B - 1))
  h0, dhT, dh = rnd(B, D, seed=3), rnd(B, D, seed=4), rnd(B * T, D, seed=5, dtype=dt)
  hs, hT = Slot(B * T, D, dt, 0, 8), h0.cuda()
  kw = dict(first=first.cuda(), shift=-1.0, cand=cand)
  hip.gated_scan_fwd(u, c, hs.t, T, i=i, h0=hT, hT=hT, **kw)                   # the state in place
  h, T1 = torch.zeros(B * T, D).double(), torch.zeros(B, D).double()
  kr = dict(first=first, shift=-1.0, cand=cand)
  ref.gated_scan_fwd(host[0], host[1], h, T, i=host[2], h0=h0, hT=T1, **kr)
  # A step's a and b are off by at most 32 u of their size (an exponential, a reciprocal, a product,
  # the composition's own rounding); e[t] = a e[t-1] + 32 u (a |h[t-1]| + |b|), majorised by
  # e[t] = a e[t-1] + 32 u m[t] with m the recurrence of the magnitudes.
  _, _, a, restart, g, phi = ref._scan_gates(host[0], host[1], host[2], T, first, -1.0, cand)
  a = torch.where(restart, torch.zeros_like(a), a)
  # bf16 operands: a is 1 - z with z good to 8 u, so off by 8 u of one, and phi is 1 - 2 r with r good to
  # 8 u, off by 16 u of one: 8 u |h[t-1]| + 16 u gate more.
  low = 1.0 if dt == BF16 else 0.0
  m = linear_recurrence(a, (g * phi).abs() + U, h0.double().abs())
  mp = torch.cat([h0.double().abs()[:, None], m[:, :-1]], 1)
  e = linear_recurrence(a, 32 * U * m + low * U * (8 * mp + 16 * g), torch.zeros(B, D).double())
  within(hs.t, h, e.reshape(B * T, D), 'h')
  within(hT, T1, e[:, -1], 'hT')
  d = Slot(B * T, n * D, dt, 0, 8 if D % 8 == 0 else 1)
  outs = [d.t[:, k * D:(k + 1) * D] for k in range(n)]
  di = outs[2] if gate else None
  dh0 = dhT.cuda()
  hip.gated_scan_bwd(dh.cuda(), u, c, hs.t, outs[0], outs[1], T, i=i, di=di, h0=h0.cuda(), dhT=dh0, dh0=dh0, **kw)
  want = [torch.zeros(B * T, D).double() for _ in range(n)]
  w0 = torch.zeros(B, D).double()
  hq = hs.t.cpu()                                                              # the backward pass reads the stored h
  ref.gated_scan_bwd(dh, host[0], host[1], hq, want[0], want[1], T, i=host[2], di=want[2] if gate else None, h0=h0, dhT=dhT, dh0=w0, **kr)
  after = torch.cat([a[:, 1:], torch.ones_like(a[:, :1])], 1).flip(1)
  mg = linear_recurrence(after, dh.double().reshape(B, T, D).abs().flip(1), dhT.double().abs())
  mgn = torch.cat([dhT.double().abs()[:, None], mg[:, :-1]], 1)
  eg = linear_recurrence(after, 32 * U * mg + low * 8 * U * mgn, torch.zeros(B, D).double()).flip(1)
  mg = mg.flip(1)
  eg = eg + 64 * U * mg                                                        # and the factors below
  before = torch.cat([h0.double()[:, None], hq.double().reshape(B, T, D)[:, :-1]], 1).abs() + phi.abs()
  z = torch.sigmoid(host[0].double().reshape(B, T, D) - 1.0)
  within(outs[0], want[0], (eg * before * z * (1 - z) + low * U * mg * z * (8 * before + 16)).reshape(B * T, D), 'du')
  # 1 - tanh^2 cancels: its error is 16 u of one, not of itself
  within(outs[1], want[1], (eg * g + (16 + 32 * low) * U * mg * g).reshape(B * T, D), 'dc')
  if gate:   # 1 - sigmoid(i) the same way: 8 u of one
    within(outs[2], want[2], (eg * phi.abs() * g * (1 - g) + U * mg * g * (8 * phi.abs() + 16 * low)).reshape(B * T, D), 'di')
  within(dh0, w0, a[:, 0] * eg[:, 0] + low * 8 * U * mg[:, 0], 'dh0')
  hs.whole(), d.whole()


@pytest.mark.parametrize('B,T,D', [(300, 256, 131), (100, 704, 131), (100, 704, 129)])
@pytest.mark.parametrize('gate,cand', [(False, 'tanh'), (True, None)])
def test_scan_of_many_unaligned_rows(hip, ref, B, T, D, gate, cand):
  """Rows that share cache lines with their neighbours, enough of them for two fp32 channels per lane, the last of
  which overlap where a row is odd; whole and split."""
  test_scan(hip, ref, B, T, D, gate, cand, F32)


def test_scan_defaults(hip, ref):
  """No restarts, no initial state, no final one."""
  u, c = rnd(60, 32, seed=1), rnd(60, 32, seed=2)
  h, want = torch.zeros(60, 32, device='cuda'), torch.zeros(60, 32).double()
  hip.gated_scan_fwd(u.cuda(), c.cuda(), h, 20)
  ref.gated_scan_fwd(u, c, want, 20)
  within(h, want, 64 * U * 8.0, 'h')
  du, dc, wu, wc = (torch.zeros(60, 32, device=d, dtype=t) for d, t in [('cuda', F32)] * 2 + [('cpu', torch.float64)] * 2)
  dh = rnd(60, 32, seed=3)
  hip.gated_scan_bwd(dh.cuda(), u.cuda(), c.cuda(), h, du, dc, 20)
  ref.gated_scan_bwd(dh, u, c, h.cpu(), wu, wc, 20)
  within(du, wu, 256 * U * 8.0, 'du'), within(dc, wc, 256 * U * 8.0, 'dc')


@pytest.mark.parametrize('T,B', [(40, 3), (700, 1)])
def test_scan_in_pieces_equals_the_whole(hip, T, B):
  """A sequence fed in pieces through its state, down to single steps, gives the scan of the whole."""
  D = 96
  u, c = rnd(B * T, D, seed=1).cuda(), rnd(B * T, D, seed=2).cuda()
  first = restarts(B, T, 0.05, 3).cuda()
  h0 = rnd(B, D, seed=4).cuda()
  whole, hT = torch.zeros(B * T, D, device='cuda'), torch.zeros(B, D, device='cuda')
  hip.gated_scan_fwd(u, c, whole, T, first=first, h0=h0, hT=hT)
  state, rows = h0.clone(), []
  at = 0
  for n in [1, 1, 5, 1, T - 8]:
    pick = lambda t: t.reshape(B, T, -1)[:, at:at + n].reshape(B * n, -1).contiguous()  # noqa: E731
    out = torch.zeros(B * n, D, device='cuda')
    f = first.reshape(B, T)[:, at:at + n].reshape(-1).contiguous()
    if n == 1:
      hip.gated_step(pick(u), pick(c), out, state, state, first=f)
    else:
      hip.gated_scan_fwd(pick(u), pick(c), out, n, first=f, h0=state, hT=state)
    rows.append(out.reshape(B, n, D))
    at += n
  # the same sums in another association: states are below 8 here
  assert float((torch.cat(rows, 1).reshape(B * T, D) - whole).abs().max()) <= 512 * U * 8
  assert float((state - hT).abs().max()) <= 512 * U * 8


@pytest.mark.parametrize('T', [30, 2000])
def test_restart_cuts_whatever_came_before(hip, T):
  """NaN and infinity in the steps before a restart reach neither the states nor the gradients behind
  it; without a restart they stay, however long the sequence is."""
  D = 64
  u, c, dh = rnd(T, D, seed=1), rnd(T, D, seed=2), rnd(T, D, seed=3)
  cut = T // 2
  first = torch.zeros(T)
  first[cut] = 1
  clean, hT = torch.zeros(T, D, device='cuda'), torch.zeros(1, D, device='cuda')
  hip.gated_scan_fwd(u.cuda(), c.cuda(), clean, T, first=first.cuda(), hT=hT)
  h0 = torch.full((1, D), float('nan'))
  bad = c.clone()
  bad[3], bad[cut - 1] = float('inf'), float('nan')
  h, hT2 = torch.zeros(T, D, device='cuda'), torch.zeros(1, D, device='cuda')
  hip.gated_scan_fwd(u.cuda(), bad.cuda(), h, T, first=first.cuda(), h0=h0.cuda(), hT=hT2, cand=None)
  assert bool(torch.isnan(h[:cut]).all()) and bool(torch.isfinite(h[cut:]).all()) and bool(torch.isfinite(hT2).all())
  du, dc, dh0 = torch.zeros(T, D, device='cuda'), torch.zeros(T, D, device='cuda'), torch.zeros(1, D, device='cuda')
  hip.gated_scan_bwd(dh.cuda(), u.cuda(), bad.cuda(), h, du, dc, T, first=first.cuda(), h0=h0.cuda(), dh0=dh0, cand=None)
  assert bool(torch.isfinite(du[cut:]).all()) and bool(torch.isfinite(dc).all()) and bool(torch.isfinite(dh0).all())
  bad_dh = dh.clone()
  bad_dh[cut + 2] = float('nan')          # a NaN behind the restart stops there on its way back
  hip.gated_scan_bwd(bad_dh.cuda(), u.cuda(), c.cuda(), clean, du, dc, T, first=first.cuda(), dh0=dh0)
  assert bool(torch.isfinite(dc[:cut]).all()) and bool(torch.isnan(dc[cut:cut + 3]).all()) and bool(torch.isfinite(dh0).all())
  hip.gated_scan_fwd(u.cuda(), c.cuda(), h, T, h0=h0.cuda(), hT=hT2)
  assert bool(torch.isnan(h).all()) and bool(torch.isnan(hT2).all())


@pytest.mark.parametrize('gate', [False, True])
@pytest.mark.parametrize('T', [12, 700])
def test_a_nan_gate_is_not_lost(hip, T, gate):
  """A NaN in the update gate reaches every later state, and every earlier gradient, of its channel - and
  of no other."""
  D = 64
  for dt in (F32, BF16):
    u, c, i, dh = (rnd(T, D, seed=k, dtype=dt).cuda() for k in range(4))
    at = T // 2
    u[at, 5] = float('nan')
    h, du, dc, di = (torch.zeros(T, D, device='cuda', dtype=dt) for _ in range(4))
    hT, dh0 = torch.zeros(1, D, device='cuda'), torch.zeros(1, D, device='cuda')
    kw = dict(i=i) if gate else {}
    hip.gated_scan_fwd(u, c, h, T, hT=hT, **kw)
    clean = [k for k in range(D) if k != 5]
    assert bool(torch.isnan(h[at:, 5]).all()) and bool(torch.isfinite(h[:at, 5]).all()) and bool(torch.isfinite(h[:, clean]).all())
    assert bool(torch.isnan(hT[0, 5])) and bool(torch.isfinite(hT[0, clean]).all())
    hip.gated_scan_bwd(dh, u, c, torch.zeros_like(h), du, dc, T, dh0=dh0, **(dict(i=i, di=di) if gate else {}))
    assert bool(torch.isnan(dc[:at, 5]).all()) and bool(torch.isfinite(dc[at + 1:, 5]).all()) and bool(torch.isnan(dh0[0, 5]))
    assert bool(torch.isfinite(dc[:, clean]).all()) and bool(torch.isfinite(dh0[0, clean]).all())


def test_scan_saturated_gates(hip, ref):
  """Gates far out: a keeps or drops the state exactly as far as fp32 says, nothing overflows."""
  for v in (-200.0, -60.0, 60.0, 200.0):
    u, c = torch.full((12, 16), v), rnd(12, 16, seed=1)
    h, want = torch.zeros(12, 16, device='cuda'), torch.zeros(12, 16).double()
    h0 = rnd(2, 16, seed=2)
    hip.gated_scan_fwd(u.cuda(), c.cuda(), h, 6, h0=h0.cuda())
    ref.gated_scan_fwd(u, c, want, 6, h0=h0)
    within(h, want, 256 * U * 4.0, f'gate {v}')


def test_norm_and_scan_rows_far_apart(hip):
  """Offsets past 2^31 elements and 2^32 bytes: bit for bit the results of compact operands."""
  ld, R, C, T = (1 << 20) + 6, 4200, 40, 2100
  far = [torch.empty(R, ld, device='cuda', dtype=BF16) for _ in range(2)]
  assert far[0].numel() > 1 << 31
  near = [rnd(R, C, seed=k, dtype=BF16).cuda() for k in range(4)]
  src = [far[0][:, 50 * k + 1:50 * k + 1 + C] for k in range(4)]
  for a, b in zip(src, near):
    a.copy_(b)
  dst = [far[1][:, 50 * k + 1:50 * k + 1 + C] for k in range(4)]
  out = [torch.empty(R, C, device='cuda', dtype=BF16) for _ in range(4)]
  g = torch.ones(C, device='cuda')
  rstd = [torch.empty(R, device='cuda') for _ in range(2)]
  for (x, r, dy, dr), (y, s, ds, _), inv in ((src, dst, rstd[0]), (near, out, rstd[1])):
    hip.rms_norm_fwd(x, g, y, rstd=inv, res=r, s=s)
    hip.rms_norm_bwd(dy, s, inv, g, ds, None, dr)
  assert torch.equal(rstd[0], rstd[1]) and all(torch.equal(a, b) for a, b in zip(dst[:3], out[:3]))
  for (u, c, i, dh), (h, du, dc, di) in ((src, dst), (near, out)):
    hip.gated_scan_fwd(u, c, h, T, i=i)
    hip.gated_scan_bwd(dh, u, c, h, du, dc, T, i=i, di=di)
  assert all(torch.equal(a, b) for a, b in zip(dst, out))


# ---- together -------------------------------------------------------------------------------------


class Block:
  """norm -> product (update | candidate) -> scan -> product + residual stream, and back."""

  def __init__(self, ops, B, T, C, D, seed=0):
    self.ops, self.B, self.T, self.C, self.D = ops, B, T, C, D
    R, dev = B * T, 'cuda'
    e = lambda *s, t=BF16: torch.zeros(*s, device=dev, dtype=t)  # noqa: E731
    self.gamma = (1 + rnd(C, seed=seed, scale=0.1)).cuda()
    self.w1, self.b1 = rnd(2 * D, C, seed=seed + 1, scale=C ** -0.5, dtype=BF16).cuda(), rnd(2 * D, seed=seed + 2, scale=0.1).cuda()
    self.w2 = rnd(C, D, seed=seed + 3, scale=D ** -0.5, dtype=BF16).cuda()
    self.s, self.y, self.rstd, self.parts, self.h, self.out = e(R, C, t=F32), e(R, C), e(R, t=F32), e(R, 2 * D), e(R, D), e(R, C, t=F32)
    self.hT = e(B, D, t=F32)
    self.dstream, self.dout, self.dh, self.dparts, self.dy = e(R, C, t=F32), e(R, C), e(R, D), e(R, 2 * D), e(R, C)
    self.grads = dict(gamma=e(C, t=F32), w1=e(2 * D, C, t=F32), b1=e(2 * D, t=F32), w2=e(C, D, t=F32))

  def forward(self, x, res, first):
    D, ops = self.D, self.ops
    ops.rms_norm_fwd(x, self.gamma, self.y, rstd=self.rstd, res=res, s=self.s)
    ops.linear_fwd(self.y, self.w1, self.parts, bias=self.b1)
    ops.gated_scan_fwd(self.parts[:, :D], self.parts[:, D:], self.h, self.T, first=first, hT=self.hT)
    ops.linear_fwd(self.h, self.w2, self.out, res=self.s)

  def backward(self, dout, first):
    """dout: bf16 gradient of out; ends in dstream, the gradient of x and of the residual stream."""
    D, ops, g = self.D, self.ops, self.grads
    ops.linear_bwd(dout, self.h, self.w2, self.dh, g['w2'])
    ops.gated_scan_bwd(self.dh, self.parts[:, :D], self.parts[:, D:], self.h, self.dparts[:, :D], self.dparts[:, D:], self.T, first=first)
    ops.linear_bwd(self.dparts, self.y, self.w1, self.dy, g['w1'], g['b1'])
    self.dstream.copy_(dout)
    ops.rms_norm_bwd(self.dy, self.s, self.rstd, self.gamma, self.dstream, g['gamma'], dres=self.dstream)


def test_block_forward_and_backward(hip):
  B, T, C, D = 4, 37, 128, 192
  blk = Block(hip, B, T, C, D)
  x, res, dout = rnd(B * T, C, seed=10, dtype=BF16), rnd(B * T, C, seed=11), rnd(B * T, C, seed=12, dtype=BF16)
  first = restarts(B, T, 0.05, 13)
  blk.forward(x.cuda(), res.cuda(), first.cuda())
  blk.backward(dout.cuda(), first.cuda())
  leaves = [t.cpu().double().requires_grad_(True) for t in (x, res, blk.gamma, blk.w1, blk.b1, blk.w2)]
  xd, rd, gd, w1, b1, w2 = leaves
  s = xd + rd
  y = s * torch.rsqrt((s * s).mean(1, keepdim=True) + 1e-6) * gd
  p = y @ w1.t() + b1
  v, c = p[:, :D].reshape(B, T, D) - 1, torch.tanh(p[:, D:].reshape(B, T, D))
  keep = (1 - first.double()).reshape(B, T, 1)
  st, hs = torch.zeros(B, D).double(), []
  for t in range(T):
    z = torch.sigmoid(v[:, t])
    st = (1 - z) * keep[:, t] * st + z * c[:, t]
    hs.append(st)
  out = torch.stack(hs, 1).reshape(B * T, D) @ w2.t() + s
  want = torch.autograd.grad(out, leaves, dout.double())

  def rel(a, b):
    a, b = a.detach().cpu().double(), b.detach()
    return float((a - b).norm() / b.norm())
  # every stored bf16 tensor on the way adds at most half a step, 2^-8, in the 2-norm; the way to a
  # gradient passes at most eight of them (y, parts, h, dout's products, dh, dparts, dy and their reads),
  # and their effects are amplified by less than two (slopes and row norms of the block are below one)
  tol = 8 * 2 * 2.0 ** -8
  for a, b, what in [(blk.out, out, 'out'), (blk.hT, st, 'hT'), (blk.dstream, want[0], 'dx'), (blk.dstream, want[1], 'dres'),
                     (blk.grads['gamma'], want[2], 'gamma'), (blk.grads['w1'], want[3], 'w1'), (blk.grads['b1'], want[4], 'b1'),
                     (blk.grads['w2'], want[5], 'w2')]:
    assert rel(a, b) <= tol, (what, rel(a, b))


def test_block_step_by_step_equals_the_sequence(hip):
  """Serving: single steps with the carried state against the scan of the whole sequence (both bf16 rows,
  the state in fp32)."""
  B, T, C, D = 3, 12, 128, 64
  whole, step = Block(hip, B, T, C, D, seed=3), Block(hip, B, 1, C, D, seed=3)
  x, res = rnd(B * T, C, seed=20, dtype=BF16).cuda(), rnd(B * T, C, seed=21).cuda()
  whole.forward(x, res, None)
  state = torch.zeros(B, D, device='cuda')
  for t in range(T):
    rows = torch.arange(B, device='cuda') * T + t
    hip.rms_norm_fwd(x[rows], step.gamma, step.y, res=res[rows], s=step.s)
    hip.linear_fwd(step.y, step.w1, step.parts, bias=step.b1)
    hip.gated_step(step.parts[:, :D], step.parts[:, D:], step.h, state, state)
    hip.linear_fwd(step.h, step.w2, step.out, res=step.s)
    # sums of another order may round a bf16 value to its neighbour (one step, 2^-7): on the way to out
    # that is y, parts and h, of sizes up to 4, through rows of w1, w2 of norm about one
    assert float((step.out - whole.out[rows]).abs().max()) <= 3 * 2.0 ** -7 * 4
  assert float((state - whole.hT).abs().max()) <= 3 * 2.0 ** -7 * 4


def test_block_replays_from_a_graph(hip):
  """Captured once (kernel launches only: the library refuses anything else), replayed between eager work
  and synchronizations: every replay equals the eager run bit for bit, with the inputs of the moment."""
  from daydreamer_amd import graphs
  B, T, C, D = 2, 300, 128, 64
  blk = Block(hip, B, T, C, D)
  first = restarts(B, T, 0.02, 1).cuda()
  x, res, dout = rnd(B * T, C, seed=2, dtype=BF16).cuda(), rnd(B * T, C, seed=3).cuda(), rnd(B * T, C, seed=4, dtype=BF16).cuda()
  st = graphs.stream('cuda:0', 'block-test')
  lib, ex, nodes = hip.lib, ctypes.c_void_p(), ctypes.c_int()
  blk.forward(x, res, first)
  blk.backward(dout, first)
  torch.cuda.synchronize()
  with torch.cuda.stream(st):
    # (dstream.copy_ of the backward pass converts types: a kernel, not a copy node)
    assert lib.dd_graph_capture_begin(st.cuda_stream) == 0
    blk.forward(x, res, first)
    blk.backward(dout, first)
    rc = lib.dd_graph_capture_end(st.cuda_stream, ctypes.byref(ex), ctypes.byref(nodes))
  assert rc == 0, lib.dd_last_error()
  eager = Block(hip, B, T, C, D)
  for k in range(4):
    x.copy_(rnd(B * T, C, seed=30 + k, dtype=BF16))
    eager.forward(x, res, first)
    eager.backward(dout, first)
    torch.cuda.synchronize()
    assert lib.dd_graph_launch(ex, st.cuda_stream) == 0
    torch.cuda.synchronize()
    for a, b in [(blk.out, eager.out), (blk.hT, eager.hT), (blk.dstream, eager.dstream)] + [(blk.grads[n], eager.grads[n]) for n in blk.grads]:
      assert torch.equal(a, b), k
  assert lib.dd_graph_destroy(ex) == 0


def test_two_graphs_replay_at_once(hip):
  """Two captured blocks (a split scan and split products among their launches) with a HipOps, that is a
  workspace, each, replayed at the same time on two streams with eager work between: the eager results."""
  from daydreamer_amd import graphs, hipops
  B, T, C, D = 1, 2000, 128, 64
  lib, runs = hip.lib, []
  for n in range(2):
    ops = hipops.HipOps('cuda:0')
    blk = Block(ops, B, T, C, D, seed=7 * n)
    x, res, dout = rnd(B * T, C, seed=2 + n, dtype=BF16).cuda(), rnd(B * T, C, seed=3 + n).cuda(), rnd(B * T, C, seed=4 + n, dtype=BF16).cuda()
    first = restarts(B, T, 0.01, n).cuda()
    blk.forward(x, res, first)
    blk.backward(dout, first)
    torch.cuda.synchronize()
    st, ex, nodes = graphs.stream('cuda:0', f'block-test-{n}'), ctypes.c_void_p(), ctypes.c_int()
    with torch.cuda.stream(st):
      assert lib.dd_graph_capture_begin(st.cuda_stream) == 0
      blk.forward(x, res, first)
      blk.backward(dout, first)
      assert lib.dd_graph_capture_end(st.cuda_stream, ctypes.byref(ex), ctypes.byref(nodes)) == 0, lib.dd_last_error()
    runs.append((blk, x, res, dout, first, st, ex, Block(hip, B, T, C, D, seed=7 * n)))
  for k in range(3):
    for n, (blk, x, res, dout, first, st, ex, eager) in enumerate(runs):
      x.copy_(rnd(B * T, C, seed=50 + 2 * k + n, dtype=BF16))
      eager.forward(x, res, first)
      eager.backward(dout, first)
    torch.cuda.synchronize()
    for run in runs:
      assert lib.dd_graph_launch(run[6], run[5].cuda_stream) == 0
    torch.cuda.synchronize()
    for blk, eager in ((run[0], run[7]) for run in runs):
      for a, b in [(blk.out, eager.out), (blk.hT, eager.hT), (blk.dstream, eager.dstream)] + [(blk.grads[m], eager.grads[m]) for m in blk.grads]:
        assert torch.equal(a, b), k
  for run in runs:
    assert lib.dd_graph_destroy(run[6]) == 0


def test_block_on_another_stream(hip):
  """The operators run on the stream that is current, in its order."""
  B, T, C, D = 2, 50, 128, 64
  a, b = Block(hip, B, T, C, D), Block(hip, B, T, C, D)
  x, res, first = rnd(B * T, C, seed=2, dtype=BF16).cuda(), rnd(B * T, C, seed=3).cuda(), restarts(B, T, 0.1, 4).cuda()
  a.forward(x, res, first)
  torch.cuda.synchronize()
  side = torch.cuda.Stream()
  with torch.cuda.stream(side):
    late = torch.zeros_like(x)
    torch.cuda._sleep(20_000_000)       # the input is written behind a delay on the side stream
    late.copy_(x)
    b.forward(late, res, first)
  side.synchronize()
  assert torch.equal(a.out, b.out)


def test_equal_calls_give_equal_bits(hip):
  B, T, C, D = 3, 700, 256, 128
  blk = Block(hip, B, T, C, D)
  x, res, first = rnd(B * T, C, seed=2, dtype=BF16).cuda(), rnd(B * T, C, seed=3).cuda(), restarts(B, T, 0.01, 4).cuda()
  dout = rnd(B * T, C, seed=5, dtype=BF16).cuda()
  got = []
  for _ in range(2):
    blk.forward(x, res, first)
    blk.backward(dout, first)
    got.append([t.clone() for t in (blk.out, blk.dstream, *blk.grads.values())])
  assert all(torch.equal(a, b) for a, b in zip(*got))


# ---- refusals of the binding ----------------------------------------------------------------------


def test_binding_refusals(hip):
  x, w = torch.zeros(4, 16, device='cuda', dtype=BF16), torch.zeros(8, 16, device='cuda', dtype=BF16)
  y, g = torch.zeros(4, 8, device='cuda', dtype=BF16), torch.zeros(16, device='cuda')
  n = torch.zeros(4, 16, device='cuda')
  calls = [
      lambda: hip.linear_fwd(x.float(), w.float(), y),                       # fp32 operands
      lambda: hip.linear_fwd(x, w.t().contiguous(), y),                      # another shape
      lambda: hip.linear_fwd(x, w.cpu(), y),                                 # another device
      lambda: hip.linear_fwd(x, w, y, res=torch.zeros(4, 8, device='cuda')), # another type than y
      lambda: hip.linear_fwd(x, w, y, bias=torch.zeros(7, device='cuda')),
      lambda: hip.linear_fwd(x.to(FP8), w.to(FP8), y),                       # no scales
      lambda: hip.linear_fwd(x[:, ::2], w[:, ::2], y),                       # strided columns
      lambda: hip.linear_fwd(x[:1].expand(4, 16), w, y),                     # broadcast rows
      lambda: hip.linear_bwd(y, x, w, dx=torch.zeros_like(x), act='silu'),   # no z
      lambda: hip.rms_norm_fwd(x, g, n, res=n),                              # nowhere to store the sum
      lambda: hip.rms_norm_fwd(x, g.to(BF16), n),
      lambda: hip.rms_norm_fwd(x, g, x.to(FP8)),                             # e4m3 without a scale
      lambda: hip.quant_rows(x, n, g[:4]),
      lambda: hip.gated_scan_fwd(x, x, n, 2),                                # h of another type
      lambda: hip.gated_scan_fwd(x, x, x.clone(), 3),                        # 4 rows are no sequences of 3
      lambda: hip.gated_scan_fwd(x, x, x.clone(), 2, first=torch.zeros(4, device='cuda', dtype=torch.bool)),
      lambda: hip.gated_scan_fwd(x, x, x.clone(), 2, cand='relu'),
      lambda: hip.gated_scan_bwd(x, x, x, x, x.clone(), x.clone(), 2, di=x.clone()),
  ]
  for k, call in enumerate(calls):
    with pytest.raises((AssertionError, RuntimeError, KeyError)):
      call()
      pytest.fail(f'call {k} was not refused')


def test_outputs_are_no_other_operands(hip):
  """Written over an operand that other workgroups still read, a result would depend on their order: refused."""
  x, w, y = torch.zeros(16, 16, device='cuda', dtype=BF16), torch.zeros(16, 16, device='cuda', dtype=BF16), torch.zeros(16, 16, device='cuda', dtype=BF16)
  a, b, g, r = torch.zeros(16, 16, device='cuda', dtype=BF16), torch.zeros(16, 16, device='cuda', dtype=BF16), torch.ones(16, device='cuda'), torch.ones(16, device='cuda')
  s0 = torch.zeros(4, 16, device='cuda')
  calls = [
      lambda: hip.linear_fwd(x, w, x),
      lambda: hip.linear_fwd(x, w, w),
      lambda: hip.linear_fwd(x, w, y, z=y),
      lambda: hip.linear_fwd(x, w, y, res=a, z=a),
      lambda: hip.linear_bwd(y, x, w, dx=x),
      lambda: hip.linear_bwd(y, x, w, dx=y),
      lambda: hip.linear_bwd(y, x, w, dw=w),
      lambda: hip.linear_bwd(y, x, w, act='silu', z=a, dz=x),
      lambda: hip.rms_norm_fwd(x, g, x),
      lambda: hip.rms_norm_bwd(y, x, r, g, x),
      lambda: hip.gated_scan_fwd(x, w, x, 4),
      lambda: hip.gated_scan_fwd(x, w, w, 4),
      lambda: hip.gated_scan_bwd(y, x, w, a, y, b, 4),
      lambda: hip.gated_scan_bwd(y, x, w, a, b, b, 4),
      lambda: hip.gated_scan_bwd(y, x, w, a, b, a, 4),
      lambda: hip.gated_scan_bwd(y, x, w, a, b, torch.zeros_like(b), 4, h0=s0, dh0=s0),
  ]
  for k, call in enumerate(calls):
    with pytest.raises(AssertionError):
      call()
      pytest.fail(f'call {k} was not refused')


def test_calls_without_rows(hip):
  """No rows: nothing is read, gradients of parameters are zero, or unchanged where they accumulate."""
  e = lambda n, t=BF16: torch.zeros(0, n, device='cuda', dtype=t)  # noqa: E731
  w, g, none = torch.ones(8, 16, device='cuda', dtype=BF16), torch.ones(16, device='cuda'), torch.zeros(0, device='cuda')
  hip.linear_fwd(e(16), w, e(8))
  hip.rms_norm_fwd(e(16), g, e(16), rstd=none)
  hip.quant_rows(e(16), e(16, FP8), none)
  hip.gated_scan_fwd(e(16), e(16), e(16), 4)
  for keep in (False, True):
    dw, db, dg = torch.full((8, 16), 3.0, device='cuda'), torch.full((8,), 3.0, device='cuda'), torch.full((16,), 3.0, device='cuda')
    hip.linear_bwd(e(8), e(16), w, dx=e(16), dw=dw, dbias=db, accumulate=keep)
    hip.rms_norm_bwd(e(16), e(16), none, g, e(16), dg, accumulate=keep)
    want = 3.0 if keep else 0.0
    assert all(bool((t == want).all()) for t in (dw, db, dg))
