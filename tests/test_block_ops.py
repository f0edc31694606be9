"""Operators of the residual recurrent block on the CPU: their float64 restatements
(oracle/ref_ops.py) against autograd and finite differences, and what the C entry points refuse
(they return before any launch, so no GPU is needed)."""

import ctypes

import pytest
import torch

from daydreamer_amd import hipops


def rnd(*shape, seed=0, scale=1.0):
  g = torch.Generator().manual_seed(seed)
  return torch.randn(*shape, generator=g, dtype=torch.float64) * scale


def same(a, b, tol=1e-12):
  assert float((a.double() - b.double()).abs().max()) <= tol * max(1.0, float(b.abs().max()))


def test_norm_restatement(ref):
  x, r, gamma, dy, dres = (rnd(*s, seed=i) for i, s in enumerate([(5, 12), (5, 12), (12,), (5, 12), (5, 12)]))
  y, s, rstd, ds, dgamma = torch.zeros(5, 12).double(), torch.zeros(5, 12).double(), torch.zeros(5).double(), torch.zeros(5, 12).double(), torch.ones(12).double()
  ref.rms_norm_fwd(x, gamma, y, rstd=rstd, res=r, s=s, eps=1e-6)
  ref.rms_norm_bwd(dy, s, rstd, gamma, ds, dgamma, dres, accumulate=True)
  leaves = [t.clone().requires_grad_(True) for t in (x, r, gamma)]
  t = leaves[0] + leaves[1]
  want = t / torch.sqrt((t * t).mean(1, keepdim=True) + 1e-6) * leaves[2]
  gx, gr, gg = torch.autograd.grad([want, t], leaves, [dy, dres])
  same(y, want.detach()), same(s, t.detach()), same(ds, gx), same(ds, gr), same(dgamma, gg + 1.0)


def test_e4m3_restatement_rounds_as_the_type():
  """Every midpoint, its neighbours and random values against torch's own conversion."""
  from oracle.ref_ops import RefOps
  codes = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()   # 0 .. 448
  mid = (codes[1:] + codes[:-1]) / 2
  v = torch.cat([codes, mid, mid * (1 + 1e-6), mid * (1 - 1e-6), rnd(5000, seed=1, scale=100.0).clamp(-448, 448)])
  v = torch.cat([v, -v])
  assert torch.equal(RefOps._e4m3(v), v.float().to(torch.float8_e4m3fn).double())


@pytest.mark.parametrize('act', [None, 'elu', 'silu', 'gelu'])
def test_linear_restatement(ref, act):
  M, N, K = 4, 5, 6
  x, w, b, r, dy = (rnd(*s, seed=i + 3) for i, s in enumerate([(M, K), (N, K), (N,), (M, N), (M, N)]))
  y, z, dz, dx, dw, db = (torch.zeros(*s).double() for s in [(M, N), (M, N), (M, N), (M, K), (N, K), (N,)])
  ref.linear_fwd(x, w, y, bias=b, act=act, res=r, z=z)
  ref.linear_bwd(dy, x, w, dx, dw, db, act=act, z=z, dz=dz)

  def f(x, w, b):
    t = x @ w.t() + b
    if act == 'elu':
      t = torch.nn.functional.elu(t)
    if act == 'silu':
      t = torch.nn.functional.silu(t)
    if act == 'gelu':
      t = torch.nn.functional.gelu(t)
    return t + r
  leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
  want = f(*leaves)
  same(y, want.detach())
  for g, t in zip(torch.autograd.grad(want, leaves, dy), (dx, dw, db)):
    same(t, g)
  d = rnd(M, K, seed=9)   # a difference quotient along one direction: error O(h^2)
  q = ((f(x + 1e-5 * d, w, b) - f(x - 1e-5 * d, w, b)) * dy).sum() / 2e-5
  assert abs(float(q - (dx * d).sum())) < 1e-7


@pytest.mark.parametrize('gate', [False, True])
@pytest.mark.parametrize('cand', ['tanh', None])
def test_scan_restatement(ref, gate, cand):
  B, T, D = 3, 7, 4
  u, c, i, dh = (rnd(B * T, D, seed=k + 20) for k in range(4))
  h0, dhT = rnd(B, D, seed=30), rnd(B, D, seed=31)
  first = torch.zeros(B, T)
  first[0, 0] = first[1, 3] = first[1, 4] = first[2, 6] = 1
  first = first.reshape(-1)
  i = i if gate else None
  h, hT, dh0 = torch.zeros(B * T, D).double(), torch.zeros(B, D).double(), torch.zeros(B, D).double()
  grads = [torch.zeros(B * T, D).double() for _ in range(3 if gate else 2)]
  ref.gated_scan_fwd(u, c, h, T, i=i, first=first, h0=h0, hT=hT, shift=-0.7, cand=cand)
  ref.gated_scan_bwd(dh, u, c, h, grads[0], grads[1], T, i=i, di=grads[2] if gate else None, first=first, h0=h0,
                     dhT=dhT, dh0=dh0, shift=-0.7, cand=cand)

  def f(u, c, h0, i=None):
    x, out = h0, []
    for t in range(T):
      z = torch.sigmoid(u.reshape(B, T, D)[:, t] - 0.7)
      m = 1 - first.reshape(B, T, 1)[:, t].double()
      v = c.reshape(B, T, D)[:, t]
      g = z if i is None else torch.sigmoid(i.reshape(B, T, D)[:, t])
      x = (1 - z) * m * x + g * (torch.tanh(v) if cand else v)
      out.append(x)
    return torch.stack(out, 1).reshape(B * T, D), x
  leaves = [t.clone().requires_grad_(True) for t in ([u, c, h0, i] if gate else [u, c, h0])]
  wh, wT = f(*leaves)
  same(h, wh.detach()), same(hT, wT.detach())
  gu, gc, g0, *gi = torch.autograd.grad([wh, wT], leaves, [dh, dhT])
  same(grads[0], gu), same(grads[1], gc), same(dh0, g0)
  if gate:
    same(grads[2], gi[0])
  d = rnd(B, D, seed=40)
  args = [i] if gate else []
  p, m = f(u, c, h0 + 1e-5 * d, *args), f(u, c, h0 - 1e-5 * d, *args)
  q = (((p[0] - m[0]) * dh).sum() + ((p[1] - m[1]) * dhT).sum()) / 2e-5
  assert abs(float(q - (dh0 * d).sum())) < 1e-7


# ---- refusals of the C entry points ---------------------------------------------------------------

F32, BF16, E4M3 = 0, 1, 2
P = 1 << 20   # a pointer that is never followed


def refused(name, *args):
  lib = hipops.load_library()
  rc = getattr(lib, name)(*args)
  assert rc == -1, (name, rc)
  text = lib.dd_last_error().decode()
  assert text.startswith('dd_'), text
  return text


def norm_args(**k):
  a = dict(x=P, ldx=8, xt=BF16, r=P, ldr=8, rt=F32, s=P, lds=8, g=P, y=P, ldy=8, yt=BF16, rstd=P, scale=None, rows=2, C=8,
           eps=1e-6, st=None)
  a.update(k)
  return list(a.values())


@pytest.mark.parametrize('change,word', [
    (dict(C=0), 'C > 0'), (dict(rows=-1), 'rows >= 0'), (dict(x=None), 'null'), (dict(g=None), 'null'), (dict(ldx=7), 'leading'),
    (dict(ldr=7), 'leading'), (dict(s=None), 'res without s'), (dict(xt=E4M3), 'fp32 or bf16'), (dict(rt=E4M3), 'fp32 or bf16'),
    (dict(yt=3), 'e4m3'), (dict(yt=E4M3), 'scale'), (dict(scale=P), 'scale'),
    (dict(C=40000, ldx=40000, ldr=40000, lds=40000, ldy=40000), '32768')])
def test_norm_refusals(change, word):
  assert word in refused('dd_rms_norm_fwd', *norm_args(**change))


def test_norm_backward_refusals():
  def args(**k):
    a = dict(dy=P, ldy=8, yt=BF16, s=P, lds=8, rt=F32, rstd=P, g=P, dres=P, ldr=8, ds=P, ldd=8, dg=P, acc=0, rows=2, C=8,
             ws=P, n=1 << 20, st=None)
    a.update(k)
    return list(a.values())
  for change, word in [(dict(C=0), 'C > 0'), (dict(dy=None), 'null'), (dict(ldd=4), 'leading'), (dict(yt=E4M3), 'bf16'),
                       (dict(n=16), 'workspace')]:
    assert word in refused('dd_rms_norm_bwd', *args(**change))


def test_quant_refusals():
  for args, word in [((P, 8, E4M3, P, 8, P, 2, 8, None), 'bf16'), ((P, 8, BF16, P, 8, None, 2, 8, None), 'null'),
                     ((P, 8, BF16, P, 7, P, 2, 8, None), 'leading'), ((P, 8, BF16, P, 8, P, 2, 0, None), 'C > 0')]:
    assert word in refused('dd_quant_rows', *args)


def test_linear_refusals():
  def args(**k):
    a = dict(x=P, ldx=16, w=P, ldw=16, type=BF16, xs=None, ws_=None, bias=P, act=0, res=None, ldr=0, y=P, ldy=8, yt=BF16, z=None,
             ldz=0, M=4, N=8, K=16, ws=P, n=1 << 20, st=None)
    a.update(k)
    return list(a.values())
  for change, word in [(dict(K=0), 'K > 0'), (dict(N=0), 'N > 0'), (dict(M=-1), 'M >= 0'), (dict(type=F32), 'dd_gemm_f32'),
                       (dict(yt=E4M3), 'bf16 or fp32'), (dict(act=9), 'activation'), (dict(type=E4M3), 'scale'),
                       (dict(xs=P), 'scale'), (dict(x=None), 'null'), (dict(ldx=15), 'leading'), (dict(ldy=7), 'leading'),
                       (dict(res=P, ldr=7), 'leading'), (dict(z=P, ldz=7), 'leading')]:
    assert word in refused('dd_linear_fwd', *args(**change))
  assert 'null' in refused('dd_linear_bwd_data', None, 8, P, 16, P, 16, BF16, 4, 8, 16, P, 1 << 20, None)
  assert 'leading' in refused('dd_linear_bwd_data', P, 7, P, 16, P, 16, BF16, 4, 8, 16, P, 1 << 20, None)
  assert 'bf16 or fp32' in refused('dd_linear_bwd_weight', P, 8, P, 16, P, 16, E4M3, 0, 4, 8, 16, P, 1 << 20, None)
  assert 'leading' in refused('dd_linear_bwd_weight', P, 8, P, 16, P, 15, BF16, 0, 4, 8, 16, P, 1 << 20, None)
  assert 'z and dz' in refused('dd_linear_act_bwd', P, 8, None, 0, 2, P, 8, P, F32, 0, 4, 8, P, 1 << 20, None)
  assert 'workspace' in refused('dd_linear_act_bwd', P, 8, P, 8, 2, P, 8, P, F32, 0, 4, 8, P, 16, None)


def test_scan_refusals():
  def args(**k):
    a = dict(u=P, ldu=8, c=P, ldc=8, i=None, ldi=0, type=BF16, first=None, fs=0, h0=None, h=P, ldh=8, hT=None, B=2, T=4, D=8,
             shift=-1.0, tanh=1, ws=P, n=1 << 20, st=None)
    a.update(k)
    return list(a.values())
  for change, word in [(dict(T=0), 'T'), (dict(D=0), 'D'), (dict(B=-1), 'B >= 0'), (dict(type=E4M3), 'fp32 or bf16'),
                       (dict(u=None), 'null'), (dict(ldc=7), 'leading'), (dict(i=P, ldi=7), 'leading'),
                       (dict(T=4096, n=64), 'workspace')]:
    assert word in refused('dd_gated_scan_fwd', *args(**change))
  tail = (P, 8, BF16, None, 0, None, None, P, 8, P, 8)
  more = (None, 2, 4, 8, -1.0, 1, P, 1 << 20, None)
  assert 'di goes with i' in refused('dd_gated_scan_bwd', P, 8, P, 8, P, 8, P, 8, *tail, None, 0, *more)
  assert 'null' in refused('dd_gated_scan_bwd', None, 8, P, 8, P, 8, None, 0, *tail, None, 0, *more)


def test_native_binding_refuses_before_it_calls():
  """The checks of daydreamer_amd._block come before any launch: tensors of the host, other types and
  wrong argument counts raise, and nothing is followed."""
  hipops.load_library()
  from daydreamer_amd import _block
  x, g = torch.zeros(2, 8), torch.zeros(8)
  with pytest.raises(AssertionError, match='x is not on device 0'):
    _block.rms_norm_fwd(0, 0, x, g, x.clone(), None, None, None, None, 1e-6)
  with pytest.raises(AssertionError, match='not on device'):
    _block.linear_fwd(0, 0, x.bfloat16(), x.bfloat16(), x, None, None, None, None, None, None, 0, 0)
  with pytest.raises(AssertionError, match='x is no tensor'):
    _block.quant_rows(0, 0, 3, x, g)
  with pytest.raises(AssertionError, match='2 rows are no sequences of 3 steps'):
    _block.gated_scan_fwd(0, 0, x, x, x, 3, None, None, None, None, -1.0, 'tanh', 0, 0)
  with pytest.raises(AssertionError, match='has 1 axes'):
    _block.rms_norm_bwd(0, 0, g, g, g, g, g, None, None, 0, 0, 0)
  with pytest.raises(AssertionError, match='arguments are needed'):
    _block.linear_bwd(0, 0, x)
  with pytest.raises(TypeError):
    _block.gated_scan_fwd(0, 0, x, x, x, 'T', None, None, None, None, -1.0, 'tanh', 0, 0)


def test_empty_calls_do_nothing():
  lib = hipops.load_library()
  assert lib.dd_rms_norm_fwd(*norm_args(rows=0, x=None, y=None)) == 0
  assert lib.dd_quant_rows(None, 8, BF16, None, 8, None, 0, 8, None) == 0
  assert lib.dd_linear_fwd(None, 16, P, 16, BF16, None, None, None, 0, None, 0, None, 8, BF16, None, 0, 0, 8, 16, P, 64, None) == 0
  assert lib.dd_linear_bwd_data(None, 8, P, 16, None, 16, BF16, 0, 8, 16, P, 64, None) == 0
  assert lib.dd_linear_bwd_weight(None, 8, None, 16, P, 16, BF16, 1, 0, 8, 16, P, 64, None) == 0
  assert lib.dd_gated_scan_fwd(None, 8, None, 8, None, 0, BF16, None, 0, None, None, 8, None, 0, 4, 8, -1.0, 1, P, 64, None) == 0
