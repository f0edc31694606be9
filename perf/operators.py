"""Measured cases of the operators of a residual recurrent block.

The block is what a sequence model of latents is stacked from: a root-mean-square norm that also adds
the residual stream, a matrix product with its bias, activation and residual in the epilogue (bf16, or
e4m3 with a scale per row for serving), and a gated recurrence that is linear in its state, so that all
time steps of a replayed sequence are one scan.  `listed` has the cases with fixed sizes, `draw` makes
more of the same ranges, `prepare` the inputs and the caller-owned output buffers, and `run` makes one
pass: in plain torch, or with `own` set through `daydreamer_amd.hipops.HipOps`.

Definitions (rows of a sequence batch are b * T + t, D channels):

  norm     s = round(x + res);  y = s * rsqrt(mean(s^2) + EPS) * gamma;  the 8-bit form divides a row of y by
           scale = max|y| / 448 and rounds to e4m3
  linear   z = x @ w^T * (row scales) + bias;  y = act(z) + res
  scan     v = u + SHIFT;  a = sigmoid(-v), 0 where the sequence starts anew;  b = sigmoid(v) * tanh(c), or
           sigmoid(i) * tanh(c) with an input gate;  h[t] = a[t] * h[t-1] + b[t]
"""

import math

import torch

own = False

EPS = 1e-6
SHIFT = -1.0
E4M3_MAX = 448.0
TYPES = {'bf16': torch.bfloat16, 'fp32': torch.float32}
_hip = []


def _ops():
  if not _hip:
    from daydreamer_amd import hipops
    _hip.append(hipops.HipOps('cuda:0'))
  return _hip[0]


# ---- cases ----------------------------------------------------------------------------------------


def listed():
  return [
      # eight environments' next step through the norm of a 1024-wide stream: latency
      dict(name='norm_step', op='norm', rows=8, cols=1024, x='bf16', res='fp32', train=False),
      # a replay minibatch (50 sequences x 50 steps) in training
      dict(name='norm_replay', op='norm', rows=2500, cols=1024, x='bf16', res='fp32', train=True),
      # feature rows deter 512 + stoch 1024 + 6 actions: rows that are no multiple of 16 bytes
      dict(name='norm_features', op='norm', rows=20001, cols=1542, x='bf16', res='bf16', train=True),
      # serving: norm to e4m3 and the widening product that reads it
      dict(name='norm_e4m3_product', op='norm_linear', rows=16384, cols=1024, out=4096, act='gelu'),
      # 64 environments' next step of the recurrence: latency
      dict(name='scan_step', op='scan', batch=64, time=1, width=1024, x='bf16', gate=False, train=False),
      # a replay minibatch in training, sequences that restart inside the chunk
      dict(name='scan_replay', op='scan', batch=50, time=50, width=1024, x='bf16', gate=False, train=True),
      # the wide model's shard (deter 4096)
      dict(name='scan_wide', op='scan', batch=32, time=64, width=4096, x='bf16', gate=True, train=True),
      # two long episodes: few channels, so the time axis has to be split
      dict(name='scan_long', op='scan', batch=2, time=16385, width=512, x='fp32', gate=True, train=True),
      # eight environments' next step through the product that makes gate and candidate: reads the weights
      dict(name='linear_step', op='linear', rows=8, out=2048, inp=1024, act='none', res=False, train=False, wide=False),
      # a replay minibatch in training, input rows that are no multiple of 16 bytes
      dict(name='linear_features', op='linear', rows=2500, out=2048, inp=1542, act='silu', res=False, train=True, wide=False),
      # the imagined trajectory (2500 starts x 15 steps) through an output product with its residual
      dict(name='linear_imagined', op='linear', rows=37500, out=1024, inp=2048, act='none', res=True, train=True, wide=True),
      # serving: rows quantised to e4m3, then the output product with its residual
      dict(name='linear_e4m3_step', op='quant_linear', rows=32, out=1024, inp=4096, act='none'),
  ]


MOST = 37500 * 1024 * 2048


def _log(rng, lo, hi):
  return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
  """Mostly multiples of 64, as layers are sized, and odd ones among them."""
  n = _log(rng, lo, hi)
  return n if rng.random() < 0.35 else max(64, n // 64 * 64)


def draw(rng):
  op = rng.choice(['norm', 'norm_linear', 'scan', 'scan', 'linear', 'linear', 'quant_linear'])
  if op == 'norm':
    cols = _width(rng, 64, 8192)
    rows = _log(rng, 1, min(40000, 60_000_000 // cols))
    x = rng.choice(['bf16', 'fp32'])
    return dict(op=op, rows=rows, cols=cols, x=x, res='fp32' if x == 'fp32' else rng.choice(['bf16', 'fp32']),
                train=rng.random() < 0.6)
  if op == 'norm_linear':
    cols, out = _width(rng, 128, 4096), _width(rng, 128, 4096)
    return dict(op=op, rows=_log(rng, 1, min(32768, MOST // (cols * out))), cols=cols, out=out,
                act=rng.choice(['none', 'elu', 'silu', 'gelu']))
  if op == 'scan':
    width = _width(rng, 64, 4096)
    time = _log(rng, 1, 32768)
    batch = _log(rng, 1, max(1, min(256, 17_000_000 // (width * time))))
    return dict(op=op, batch=batch, time=time, width=width, x=rng.choice(['bf16', 'fp32']),
                gate=rng.random() < 0.5, train=time > 1 and rng.random() < 0.6)
  inp, out = _width(rng, 64, 4096), _width(rng, 64, 4096)
  rows = _log(rng, 1, min(40000, MOST // (inp * out)))
  act = rng.choice(['none', 'elu', 'silu', 'gelu'])
  if op == 'quant_linear':
    return dict(op=op, rows=rows, out=out, inp=inp, act=act)
  return dict(op=op, rows=rows, out=out, inp=inp, act=act, res=rng.random() < 0.5, train=rng.random() < 0.6,
              wide=act == 'none' and rng.random() < 0.5)


# ---- inputs ---------------------------------------------------------------------------------------


def prepare(case, seed):
  dev = 'cuda'
  g = torch.Generator(device=dev).manual_seed(seed)

  def normal(*shape, scale=1.0, dtype=torch.float32):
    return torch.empty(shape, device=dev).normal_(0.0, scale, generator=g).to(dtype)

  def empty(*shape, dtype=torch.float32):
    return torch.empty(shape, device=dev, dtype=dtype)

  s = dict(case)
  if case['op'] in ('norm', 'norm_linear'):
    rows, cols = case['rows'], case['cols']
    xt, rt = TYPES[case.get('x', 'bf16')], TYPES[case.get('res', 'fp32')]
    s.update(x=normal(rows, cols, dtype=xt), res=normal(rows, cols, scale=2.0, dtype=rt),
             gamma=1.0 + normal(cols, scale=0.1), s=empty(rows, cols, dtype=rt), rstd=empty(rows))
    if case['op'] == 'norm':
      s.update(y=empty(rows, cols, dtype=xt))
      if case['train']:
        s.update(dy=normal(rows, cols, dtype=xt), dres=normal(rows, cols, dtype=rt),
                 ds=empty(rows, cols, dtype=rt), dgamma=empty(cols))
      return s
  if case['op'] == 'scan':
    B, T, D = case['batch'], case['time'], case['width']
    xt = TYPES[case['x']]
    n = 3 if case['gate'] else 2
    parts = normal(B * T, n * D, dtype=xt)   # one product's output: update | candidate (| input gate)
    first = (torch.rand(B, T, device=dev, generator=g) < 1 / 40).float()
    s.update(u=parts[:, :D], c=parts[:, D:2 * D], i=parts[:, 2 * D:] if case['gate'] else None,
             first=first.reshape(-1), h0=normal(B, D, scale=0.5), h=empty(B * T, D, dtype=xt), hT=empty(B, D))
    if case['train']:
      d = empty(B * T, n * D, dtype=xt)
      s.update(dh=normal(B * T, D, dtype=xt), dhT=normal(B, D), du=d[:, :D], dc=d[:, D:2 * D],
               di=d[:, 2 * D:] if case['gate'] else None, dh0=empty(B, D), d=d)
    return s
  rows, out, inp = case['rows'], case['out'], case.get('inp', case.get('cols'))
  w = normal(out, inp, scale=inp ** -0.5)
  s.update(bias=normal(out, scale=0.1))
  if case['op'] == 'linear':
    bf = torch.bfloat16
    s.update(x=normal(rows, inp, dtype=bf), w=w.to(bf), y=empty(rows, out, dtype=bf),
             res_in=normal(rows, out, dtype=bf) if case['res'] else None)
    if case['train']:
      pt = torch.float32 if case['wide'] else bf
      act = case['act'] != 'none'
      s.update(z=empty(rows, out, dtype=bf) if act else None, dz=empty(rows, out, dtype=bf) if act else None,
               dy=normal(rows, out, dtype=bf), dx=empty(rows, inp, dtype=bf), dw=empty(out, inp, dtype=pt),
               dbias=empty(out, dtype=pt))
    return s
  # e4m3: the weights are quantised once, a scale per output
  ws = w.abs().amax(1) / E4M3_MAX
  s.update(w=(w / ws[:, None]).to(torch.float8_e4m3fn), w_scale=ws, y=empty(rows, out, dtype=torch.bfloat16),
           q=empty(rows, inp, dtype=torch.float8_e4m3fn), x_scale=empty(rows))
  if case['op'] == 'quant_linear':
    s.update(x=normal(rows, inp, dtype=torch.bfloat16), res_in=normal(rows, out, dtype=torch.bfloat16))
  else:
    s.update(res_in=None)
  return s


# ---- one pass -------------------------------------------------------------------------------------


def run(s):
  if s['op'] == 'norm':
    return _norm(s)
  if s['op'] == 'scan':
    return _scan(s)
  if s['op'] == 'linear':
    return _linear(s)
  return _quantised(s)


def _norm(s):
  if own:
    ops = _ops()
    ops.rms_norm_fwd(s['x'], s['gamma'], s['y'], rstd=s['rstd'], res=s['res'], s=s['s'], eps=EPS)
    if not s['train']:
      return {'y': s['y'], 's': s['s']}
    ops.rms_norm_bwd(s['dy'], s['s'], s['rstd'], s['gamma'], s['ds'], dgamma=s['dgamma'], dres=s['dres'])
    return {'y': s['y'], 's': s['s'], 'ds': s['ds'], 'dgamma': s['dgamma']}
  y, total, rstd = _plain_norm(s['x'], s['res'], s['gamma'])
  if not s['train']:
    return {'y': y.to(s['x'].dtype), 's': total}
  n = total.float() * rstd
  dy = s['dy'].float()
  dn = dy * s['gamma']
  ds = s['dres'].float() + rstd * (dn - n * (dn * n).mean(1, keepdim=True))
  return {'y': y.to(s['x'].dtype), 's': total, 'ds': ds.to(s['res'].dtype), 'dgamma': (dy * n).sum(0)}


def _plain_norm(x, res, gamma):
  total = (x.float() + res.float()).to(res.dtype)
  t = total.float()
  rstd = torch.rsqrt((t * t).mean(1, keepdim=True) + EPS)
  return t * rstd * gamma, total, rstd


def _scan(s):
  T, gate = s['time'], s['gate']
  if own:
    ops = _ops()
    if T == 1:
      ops.gated_step(s['u'], s['c'], s['h'], s['h0'], s['hT'], i=s['i'], first=s['first'], shift=SHIFT)
    else:
      ops.gated_scan_fwd(s['u'], s['c'], s['h'], T, i=s['i'], first=s['first'], h0=s['h0'], hT=s['hT'], shift=SHIFT)
    if not s['train']:
      return {'h': s['h'], 'hT': s['hT']}
    ops.gated_scan_bwd(s['dh'], s['u'], s['c'], s['h'], s['du'], s['dc'], T, i=s['i'], di=s['di'],
                       first=s['first'], h0=s['h0'], dhT=s['dhT'], dh0=s['dh0'], shift=SHIFT)
    return {'h': s['h'], 'hT': s['hT'], 'd': s['d'], 'dh0': s['dh0']}
  B, D, xt = s['batch'], s['width'], s['u'].dtype
  view = lambda t: t.float().reshape(B, T, D)  # noqa: E731
  keep = 1.0 - s['first'].reshape(B, T, 1)
  v = view(s['u']) + SHIFT
  z = torch.sigmoid(v)
  keep_a = torch.sigmoid(-v)
  a = keep_a * keep
  cand = torch.tanh(view(s['c']))
  gi = torch.sigmoid(view(s['i'])) if gate else z
  h = _plain_scan(a, gi * cand, s['h0'])
  out = {'h': h.to(xt).reshape(B * T, D), 'hT': h[:, -1].clone()}
  if not s['train']:
    return out
  # g[t] = dh[t] + a[t+1] g[t+1]: the same scan from the end
  dh = view(s['dh'])
  after = torch.cat([torch.ones_like(a[:, :1]), a[:, 1:].flip(1)], 1)
  g = _plain_scan(after, dh.flip(1), s['dhT']).flip(1)
  before = torch.cat([s['h0'][:, None], h[:, :-1]], 1) * keep
  if gate:
    du = -g * before * z * keep_a
    di = g * cand * gi * (1.0 - gi)
  else:
    du = g * (cand - before) * z * keep_a
  dc = g * gi * (1.0 - cand * cand)
  d = torch.cat([du, dc, di] if gate else [du, dc], 2)
  return {**out, 'd': d.to(xt).reshape(B * T, -1), 'dh0': a[:, 0] * g[:, 0]}


def _plain_scan(a, b, start):
  """h[t] = a[t] h[t-1] + b[t] along axis 1 by doubling: log2(T) passes over all steps."""
  b = torch.cat([b[:, :1] + a[:, :1] * start[:, None], b[:, 1:]], 1)
  n, T = 1, a.shape[1]
  while n < T:
    b = torch.cat([b[:, :n], b[:, n:] + a[:, n:] * b[:, :-n]], 1)
    a = torch.cat([a[:, :n], a[:, n:] * a[:, :-n]], 1)
    n *= 2
  return b


def _plain_act(z, act):
  """The activation and its derivative."""
  if act == 'none':
    return z, torch.ones_like(z)
  if act == 'elu':
    e = torch.exp(torch.clamp(z, max=0.0))
    return torch.where(z > 0, z, torch.expm1(torch.clamp(z, max=0.0))), torch.where(z > 0, torch.ones_like(z), e)
  if act == 'silu':
    p = torch.sigmoid(z)
    return z * p, p * (1.0 + z * (1.0 - p))
  p = 0.5 * (1.0 + torch.erf(z * 0.5 ** 0.5))
  return z * p, p + z * torch.exp(-0.5 * z * z) * (2.0 * math.pi) ** -0.5


def _linear(s):
  act = s['act']
  if own:
    ops = _ops()
    if not s['train']:
      ops.linear_fwd(s['x'], s['w'], s['y'], bias=s['bias'], act=act, res=s['res_in'])
      return {'y': s['y']}
    ops.linear_fwd(s['x'], s['w'], s['y'], bias=s['bias'], act=act, res=s['res_in'], z=s['z'])
    ops.linear_bwd(s['dy'], s['x'], s['w'], dx=s['dx'], dw=s['dw'], dbias=s['dbias'], act=act, z=s['z'], dz=s['dz'])
    return {'y': s['y'], 'dx': s['dx'], 'dw': s['dw'], 'dbias': s['dbias']}
  x, w = s['x'].float(), s['w'].float()
  z = x @ w.t() + s['bias']
  y, slope = _plain_act(z, act)
  if s['res_in'] is not None:
    y = y + s['res_in'].float()
  y = y.to(s['y'].dtype)
  if not s['train']:
    return {'y': y}
  dz = s['dy'].float() * slope
  pt = s['dw'].dtype
  return {'y': y, 'dx': (dz @ w).to(s['x'].dtype), 'dw': (dz.t() @ x).to(pt), 'dbias': dz.sum(0).to(pt)}


def _quantised(s):
  norm = s['op'] == 'norm_linear'
  if own:
    ops = _ops()
    if norm:
      ops.rms_norm_fwd(s['x'], s['gamma'], s['q'], rstd=s['rstd'], res=s['res'], s=s['s'], scale=s['x_scale'], eps=EPS)
    else:
      ops.quant_rows(s['x'], s['q'], s['x_scale'])
    ops.linear_fwd(s['q'], s['w'], s['y'], bias=s['bias'], act=s['act'], res=s['res_in'], x_scale=s['x_scale'], w_scale=s['w_scale'])
    return {'y': s['y'], 's': s['s']} if norm else {'y': s['y']}
  if norm:
    x, total, _ = _plain_norm(s['x'], s['res'], s['gamma'])
  else:
    x = s['x'].float()
  most = x.abs().amax(1, keepdim=True)
  inv = torch.where(most > 0, E4M3_MAX / most, torch.ones_like(most))
  scale = torch.where(most > 0, most / E4M3_MAX, torch.ones_like(most))
  q = torch.clamp(x * inv, -E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).float()
  z = (q @ s['w'].float().t()) * scale * s['w_scale'] + s['bias']
  y, _ = _plain_act(z, s['act'])
  if s['res_in'] is not None:
    y = y + s['res_in'].float()
  y = y.to(s['y'].dtype)
  return {'y': y, 's': total} if norm else {'y': y}


# ---- what a pass cannot do without ----------------------------------------------------------------


def work(case):
  op = case['op']
  size = lambda t: {'bf16': 2, 'fp32': 4}[t]  # noqa: E731
  if op == 'norm':
    n = case['rows'] * case['cols']
    x, r = size(case['x']), size(case['res'])
    bytes_, flops = n * (2 * x + 2 * r) + 4 * case['cols'], 5 * n
    if case['train']:   # dy, s, dres in; ds out
      bytes_ += n * (x + 3 * r) + 4 * case['cols']
      flops += 9 * n
    return dict(bytes=bytes_, flops=flops)
  if op == 'scan':
    n, e = case['batch'] * case['time'] * case['width'], size(case['x'])
    gates = 3 if case['gate'] else 2
    state = 8 * case['batch'] * case['width']
    bytes_, flops = n * e * (gates + 1) + state + 4 * case['batch'] * case['time'], 12 * n
    if case['train']:   # dh, gates, h in; the gates' gradients out
      bytes_ += n * e * (2 * gates + 2) + state
      flops += 24 * n
    return dict(bytes=bytes_, flops=flops)
  M, N, K = case['rows'], case['out'], case.get('inp', case.get('cols'))
  flops = 2.0 * M * N * K
  if op == 'linear':
    bytes_ = 2 * (M * K + N * K + M * N) + 4 * N + (2 * M * N if case['res'] else 0)
    if case['train']:
      p = 4 if case['wide'] else 2
      bytes_ += 2 * (M * N + 2 * M * K + N * K) + p * (N * K + N) + (2 * M * N if case['act'] != 'none' else 0)
      flops *= 3
    return dict(bytes=bytes_, flops=flops)
  bytes_ = 2 * M * K + N * K + 2 * M * N + 8 * N
  bytes_ += 8 * M * K + 4 * K if op == 'norm_linear' else 2 * M * N
  return dict(bytes=bytes_, flops=flops)


# ---- the definitions in 64 bits -------------------------------------------------------------------


def exact(case, seed):
  s = prepare(case, seed)
  if case['op'] == 'norm':
    return _exact_norm(s)
  if case['op'] == 'scan':
    return _exact_scan(s)
  if case['op'] == 'linear':
    return _exact_linear(s)
  return _exact_quantised(s)


def _phi(z, act):
  z = z.detach().requires_grad_(True)
  y = {'none': lambda: z * 1.0, 'elu': lambda: torch.where(z > 0, z, torch.exp(z.clamp(max=0)) - 1),
       'silu': lambda: z / (1 + torch.exp(-z)), 'gelu': lambda: z * (1 - torch.special.erfc(z / 2 ** 0.5) / 2)}[act]()
  return y.detach(), torch.autograd.grad(y.sum(), z)[0]


def _exact_norm(s):
  total = (s['x'].double() + s['res'].double()).to(s['res'].dtype)
  t = total.double().requires_grad_(True)
  gamma = s['gamma'].double().requires_grad_(True)
  y = gamma * t / torch.sqrt(t.square().sum(1, keepdim=True) / t.shape[1] + EPS)
  out = {'y': y.detach(), 's': total.double()}
  if s['train']:
    dt, dgamma = torch.autograd.grad(y, [t, gamma], s['dy'].double())
    out.update(ds=dt + s['dres'].double(), dgamma=dgamma)
  return out


def _exact_scan(s):
  """Step by step."""
  B, T, D = s['batch'], s['time'], s['width']
  u, c = (s[k].double().reshape(B, T, D) for k in ('u', 'c'))
  first = s['first'].reshape(B, T) != 0
  z = 1 / (1 + torch.exp(-SHIFT - u))
  gi = 1 / (1 + torch.exp(-s['i'].double().reshape(B, T, D))) if s['gate'] else z
  a = torch.where(first[..., None], torch.zeros_like(z), 1 / (1 + torch.exp(u + SHIFT)))
  cand = torch.tanh(c)
  b = gi * cand
  h, now = torch.empty_like(b), s['h0'].double()
  for t in range(T):
    now = torch.addcmul(b[:, t], a[:, t], now)
    h[:, t] = now
  out = {'h': h.reshape(B * T, D), 'hT': now}
  if not s['train']:
    return out
  g, now = torch.empty_like(b), s['dhT'].double()
  dh = s['dh'].double().reshape(B, T, D)
  for t in range(T - 1, -1, -1):
    now = dh[:, t] + now
    g[:, t] = now
    now = now * a[:, t]
  last = torch.cat([s['h0'].double()[:, None], h[:, :-1]], 1)
  da = torch.where(first[..., None], torch.zeros_like(last), g * last)
  slope = z - z * z
  db = g * cand
  parts = [slope * (-da), g * gi * (1 - cand ** 2), db * (gi - gi * gi)] if s['gate'] else [slope * (db - da), g * gi * (1 - cand ** 2)]
  return {**out, 'd': torch.cat(parts, 2).reshape(B * T, -1), 'dh0': now}


def _exact_linear(s):
  x, w = s['x'].double(), s['w'].double()
  y, slope = _phi(torch.addmm(s['bias'].double(), x, w.t()), s['act'])
  if s['res_in'] is not None:
    y = y + s['res_in'].double()
  if not s['train']:
    return {'y': y}
  dz = slope * s['dy'].double()
  return {'y': y, 'dx': torch.mm(dz, w), 'dw': torch.mm(dz.t(), x), 'dbias': dz.sum(0)}


def _e4m3(v):
  """Nearest e4m3 value, ties to even: three bits behind the leading one, steps of 2^-9 below 2^-6."""
  step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
  return torch.clamp(torch.round(v / step) * step, -E4M3_MAX, E4M3_MAX)


def _exact_quantised(s):
  out = {}
  if s['op'] == 'norm_linear':
    total = (s['x'].double() + s['res'].double()).to(s['res'].dtype)
    t = total.double()
    x = s['gamma'].double() * t / torch.sqrt(t.square().sum(1, keepdim=True) / t.shape[1] + EPS)
    out['s'] = t
  else:
    x = s['x'].double()
  most = x.abs().max(1, keepdim=True).values
  scale = torch.where(most > 0, most / E4M3_MAX, torch.ones_like(most))
  z = torch.mm(_e4m3(x / scale), s['w'].double().t()) * scale * s['w_scale'].double() + s['bias'].double()
  y = _phi(z, s['act'])[0]
  if s['res_in'] is not None:
    y = y + s['res_in'].double()
  return {'y': y, **out}
