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
