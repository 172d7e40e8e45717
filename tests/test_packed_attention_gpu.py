"""Rotary positions, norms of queries and keys with the rotation, and packed attention on the GPU, against
plain implementations in 64 bits.

Tolerances count roundings.  A value rounded to bf16 is off by at most half a step, HB = 2^-8 of itself, to fp32 by HF =
2^-24.  Attention: the weights P enter the matrix instruction in bf16, so |out - exact| <= HB sum_j P_j |v_j| (weights)
+ HB |out| (the result), plus the weights' own relative error rp: a score is a fp32 sum of D products, off by at most
D HF sum |q k| scale, and the exponential and the sum of the weights add some 2^-20.  Backward likewise, with the error
of delta = sum dout out (out and what its rounding left: 2^-16 of it) and of dS on its way into the matrix instruction.
"""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

HB, HF = 2.0 ** -8, 2.0 ** -24


@pytest.fixture(scope="module")
def K(dev):
  from compare_gan_amd.hip import kernels
  return kernels


@pytest.fixture(scope="module")
def Fn(dev):
  from compare_gan_amd.hip import functional
  return functional


def within(got, want, tol, what):
  got = got.double().cpu()
  bad = ~((got - want).abs() <= tol)
  if bad.any():
    i = tuple(int(x) for x in bad.nonzero()[0])
    ratio = ((got - want).abs() / tol).nan_to_num(float("inf")).max()
    raise AssertionError("%s: %d of %d off, first at %s: %r, exact %r, tolerance %r (worst ratio %.3g)" % (
        what, int(bad.sum()), got.numel(), i, float(got[i]), float(want[i]), float(tol[i]), ratio))


def normal(gen, shape, dtype=torch.bfloat16):
  return torch.randn(shape, generator=gen).to(dtype)


# ------------------------------------------------------------------------------------------------
# rotation and norm
# ------------------------------------------------------------------------------------------------
def exact_turn(x, positions, table, inverse=False):
  """x fp64 [T, H, D] on the CPU; also the sum of the magnitudes that meet in every entry."""
  rot, n = table.rotary_dim, table.rotary_dim // 2 // table.axes
  f = table.freq.cpu() * 2 * math.pi
  pos = positions.cpu().double().reshape(x.shape[0], -1)
  angle = torch.cat([pos[:, a:a + 1] * f[a * n:(a + 1) * n] for a in range(table.axes)], 1)[:, None]
  c, s = torch.cos(angle) * table.amplitude, torch.sin(angle) * table.amplitude * (-1 if inverse else 1)
  half = table.layout == "half"
  a = x[..., :rot // 2] if half else x[..., 0:rot:2]
  b = x[..., rot // 2:rot] if half else x[..., 1:rot:2]
  y, mag = x.clone(), x.abs()
  both = (a.abs() + b.abs()) * table.amplitude
  if half:
    y[..., :rot // 2], y[..., rot // 2:rot] = a * c - b * s, a * s + b * c
    mag[..., :rot // 2], mag[..., rot // 2:rot] = both, both
  else:
    y[..., 0:rot:2], y[..., 1:rot:2] = a * c - b * s, a * s + b * c
    mag[..., 0:rot:2], mag[..., 1:rot:2] = both, both
  return y, mag


def half_step(dtype):
  return HB if dtype == torch.bfloat16 else HF


# a turned entry: the angle (reduced in 64 bits, then fp32: half a step of half a turn = 2^-25 turns, 2 pi 2^-25 < 2^-22
# rad), cosine / sine (fp32 library: 2 steps; bf16 data: the hardware's, taken as good to 2^-16), three fp32 roundings
def turn_error(dtype):
  return 2.0 ** -15 if dtype == torch.bfloat16 else 2.0 ** -22 + 2 * 2.0 ** -23 + 3 * HF


ROTARY = [
    # T, H, D, rot, layout, axes, scaling, dtype
    (1, 1, 2, 2, "half", 1, "none", torch.float32),
    (1, 3, 64, 64, "half", 1, "none", torch.bfloat16),
    (7, 8, 64, 32, "interleaved", 1, "linear", torch.bfloat16),
    (130, 5, 80, 40, "half", 1, "yarn", torch.float32),
    (65, 2, 18, 10, "interleaved", 1, "ntk", torch.float32),
    (33, 3, 36, 36, "half", 3, "none", torch.bfloat16),
    (1000, 4, 128, 128, "half", 2, "yarn", torch.bfloat16),
    (19, 2, 256, 256, "half", 1, "none", torch.bfloat16),
    (19, 3, 254, 254, "interleaved", 1, "none", torch.float32),
    (5, 17, 16, 16, "half", 1, "none", torch.bfloat16),
    (4099, 1, 96, 48, "interleaved", 2, "none", torch.bfloat16),
]


def positions_of(gen, t, axes, far):
  return torch.randint(-far // 8, far, (t, axes) if axes > 1 else (t,), generator=gen, dtype=torch.int32).cuda()


@pytest.mark.parametrize("case", ROTARY, ids=[str(i) for i in range(len(ROTARY))])
def test_rotary(K, Fn, case):
  t, h, d, rot, layout, axes, scaling, dtype = case
  gen = torch.Generator().manual_seed(t + h + d)
  table = K.RotaryTable(rot, layout=layout, scaling=scaling, factor=4.0, axes=axes)
  pos = positions_of(gen, t, axes, 1 << 20)
  x = normal(gen, (t, h, d), dtype).cuda().requires_grad_(True)
  y = Fn.rotary(x, pos, table)
  want, mag = exact_turn(x.detach().double().cpu(), pos, table)
  assert y.dtype == dtype and y.shape == x.shape
  within(y, want, half_step(dtype) * want.abs() + turn_error(dtype) * mag + 1e-30, "y")
  assert torch.equal(y[..., rot:], x[..., rot:])
  dy = normal(gen, (t, h, d), dtype).cuda()
  (dx,) = torch.autograd.grad(y, (x,), dy)
  want, mag = exact_turn(dy.double().cpu(), pos, table, inverse=True)
  within(dx, want, half_step(dtype) * want.abs() + turn_error(dtype) * mag + 1e-30, "dx")


def exact_norm(x, gain, eps):
  inv = 1.0 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
  return x * inv * (1.0 if gain is None else gain)


QK = [
    # T, H, Hk, D, rot, layout, axes, dtype, merged, gains
    (1, 1, 1, 2, 2, "half", 1, torch.float32, False, True),
    (3, 4, 1, 64, 64, "half", 1, torch.bfloat16, False, True),
    (300, 6, 6, 32, 32, "half", 2, torch.bfloat16, False, True),
    (1009, 12, 4, 72, 36, "interleaved", 1, torch.bfloat16, True, True),
    (77, 3, 1, 50, 22, "half", 1, torch.float32, True, True),
    (40, 2, 2, 256, 128, "interleaved", 1, torch.bfloat16, False, False),
    (40, 2, 1, 250, 250, "half", 1, torch.float32, False, True),
    (2500, 8, 2, 128, 128, "half", 1, torch.bfloat16, True, True),
    (64, 5, 5, 16, 0, "half", 1, torch.bfloat16, False, True),
]


@pytest.mark.parametrize("case", QK, ids=[str(i) for i in range(len(QK))])
def test_qk_norm_rotary(K, Fn, case):
  t, h, hk, d, rot, layout, axes, dtype, merged, gains = case
  gen = torch.Generator().manual_seed(t + h + d)
  table = K.RotaryTable(rot, layout=layout, axes=axes) if rot else None
  pos = positions_of(gen, t, axes, 100000) if rot else None
  whole = normal(gen, (t, h + 2 * hk, d), dtype)
  whole[0] = 0.0                                   # a head of zeros: eps carries the norm
  whole = whole.cuda()
  q, k = whole[:, :h], whole[:, h:h + hk]
  if not merged:
    q, k = q.contiguous(), k.contiguous()
  q, k = q.detach().requires_grad_(True), k.detach().requires_grad_(True)
  qg = (1 + 0.3 * normal(gen, (d,), torch.float32)).cuda().requires_grad_(True) if gains else None
  kg = (1 + 0.3 * normal(gen, (d,), torch.float32)).cuda().requires_grad_(True) if gains else None
  eps = 1e-6
  qo, ko = Fn.qk_norm_rotary(q, k, qg, kg, pos, table, eps=eps)
  dqo, dko = normal(gen, q.shape, dtype).cuda(), normal(gen, k.shape, dtype).cuda()
  wanted = [x for x in (q, k, qg, kg) if x is not None]
  grads = torch.autograd.grad((qo, ko), wanted, (dqo, dko))
  te = turn_error(dtype)
  for x, g, y, dy, dx, dg in ((q, qg, qo, dqo, grads[0], grads[2] if gains else None),
                              (k, kg, ko, dko, grads[1], grads[3] if gains else None)):
    x64, g64 = x.detach().double().cpu(), (g.detach().double().cpu() if gains else None)
    n64 = exact_norm(x64, g64, eps)
    # sum of d squares, square root, divide, two products: (d + 5) fp32 roundings at most, before the turn
    rn = (d + 5) * HF
    want, mag = exact_turn(n64, pos, table) if rot else (n64, n64.abs())
    within(y, want, half_step(dtype) * want.abs() + (te + rn) * mag + 1e-30, "y")
    gy = dy.double().cpu()
    gr, gmag = exact_turn(gy, pos, table, inverse=True) if rot else (gy, gy.abs())
    inv = 1.0 / torch.sqrt(x64.square().mean(-1, keepdim=True) + eps)
    unit = x64 * inv
    gg = gr * (g64 if gains else 1.0)
    ggm = gmag * (g64.abs() if gains else 1.0)
    want = inv * (gg - unit * (gg * unit).mean(-1, keepdim=True))
    size = inv * (ggm + unit.abs() * (ggm * unit.abs()).mean(-1, keepdim=True))
    within(dx, want, half_step(dtype) * want.abs() + (te + 3 * rn) * size + 1e-30, "dx")
    if gains:
      # a fp32 sum of T heads terms in a tree of partial sums: at most (T heads) roundings of the running sum; the
      # partials of a block and the blocks' join keep it far below, the bound used is the square root of that
      rows = t * x.shape[1]
      size = (gmag * unit.abs()).sum((0, 1))
      within(dg, (gr * unit).sum((0, 1)), (te + 3 * rn + math.sqrt(rows) * HF) * size + 1e-30, "dgain")


def test_rotation_on_strided_views(K, Fn):
  """Heads and rows at any stride; a transposed head width is copied; unaligned starts take the narrow loads."""
  gen = torch.Generator().manual_seed(5)
  table = K.RotaryTable(32)
  big = normal(gen, (9, 40, 70)).cuda()
  for x in (big[:, 3:17:2, 1:65], big[::2, :5, 6:70], big[:, :, :64].transpose(0, 1), big[:, :, 2:66],
            normal(gen, (6, 64, 7)).cuda().transpose(1, 2), normal(gen, (1, 1, 64)).cuda().expand(4, 3, 64)):
    pos = positions_of(gen, x.shape[0], 1, 5000)
    want, mag = exact_turn(x.double().cpu(), pos, table)
    y = Fn.rotary(x, pos, table)
    assert y.is_contiguous()
    within(y, want, HB * want.abs() + turn_error(torch.bfloat16) * mag + 1e-30, "strided")


def test_rotation_of_nothing(K, Fn):
  table = K.RotaryTable(16)
  none = torch.empty((0,), dtype=torch.int32, device="cuda")
  x = torch.empty((0, 2, 16), dtype=torch.bfloat16, device="cuda", requires_grad=True)
  assert Fn.rotary(x, none, table).shape == (0, 2, 16)
  g = torch.ones(16, device="cuda", requires_grad=True)
  q, k = Fn.qk_norm_rotary(x, x, g, g, none, table)
  dx, dg = torch.autograd.grad((q, k), (x, g), (torch.empty_like(q), torch.empty_like(k)))
  assert dx.shape == (0, 2, 16) and torch.equal(dg, torch.zeros_like(dg))


def test_rotation_refusals(K, Fn):
  table, pos = K.RotaryTable(16, axes=2), torch.zeros((4, 2), dtype=torch.int32, device="cuda")
  x = torch.zeros((4, 2, 32), dtype=torch.bfloat16, device="cuda")
  assert Fn.rotary(x, pos, table).shape == x.shape
  for bad in (dict(x=x.half()), dict(x=x[0]), dict(x=x[..., :31]), dict(positions=pos.long()), dict(positions=pos[:3]),
              dict(positions=pos[:, 0]), dict(positions=pos.cpu()), dict(table=None), dict(x=x[..., :8]),
              dict(x=torch.zeros((4, 2, 258), dtype=torch.bfloat16, device="cuda"))):
    with pytest.raises(ValueError):
      Fn.rotary(**dict(dict(x=x, positions=pos, table=table), **bad))
  g = torch.ones(32, device="cuda")
  good = dict(q=x, k=x, q_gain=g, k_gain=None, positions=pos, table=table)
  Fn.qk_norm_rotary(**good)
  for bad in (dict(k=x.float()), dict(k=x[:3]), dict(k=x[..., :16]), dict(q_gain=g[:16]), dict(q_gain=g.double()),
              dict(positions=None), dict(eps=-1.0), dict(eps=float("nan"))):
    with pytest.raises(ValueError):
      Fn.qk_norm_rotary(**dict(good, **bad))


# ------------------------------------------------------------------------------------------------
# attention
# ------------------------------------------------------------------------------------------------
def exact_attention(q, k, v, dout, seqs, heads, kv_heads, causal, scale):
  """fp64 on the CPU: outputs, gradients and their tolerances (None entries of dout: forward only)."""
  q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
  g, d = heads // kv_heads, q.shape[2]
  out = torch.zeros(q.shape[0], heads, v.shape[2], dtype=torch.float64)
  tout = torch.full_like(out, 1e-30)
  res = {"out": (out, tout)}
  if dout is not None:
    dout = dout.double().cpu()
    for name, t in (("dq", q), ("dk", k), ("dv", v)):
      res[name] = (torch.zeros_like(t), torch.zeros_like(t))
  for q0, lq, k0, lk in seqs:
    if lq == 0 or lk == 0:
      continue
    see = torch.ones(lq, lk, dtype=torch.bool)
    if causal:
      see = torch.arange(lk)[None] <= torch.arange(lq)[:, None] + (lk - lq)
    for h in range(heads):
      a, b, c = q[q0:q0 + lq, h], k[k0:k0 + lk, h // g], v[k0:k0 + lk, h // g]
      s = (a @ b.t() * scale).masked_fill(~see, -math.inf)
      top = s.amax(-1, keepdim=True)
      p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
      p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
      o = p @ c
      rp = 2 * scale * d * HF * float((a.abs() @ b.abs().t()).max()) + 2.0 ** -20
      to = (HB + rp) * (p @ c.abs()) + HB * o.abs()
      out[q0:q0 + lq, h] = o
      tout[q0:q0 + lq, h] += to
      if dout is None:
        continue
      e = dout[q0:q0 + lq, h]
      dp = e @ c.t()
      delta = (e * o).sum(-1, keepdim=True)
      ds = p * (dp - delta)
      # dP is a fp32 sum of Dv products; delta meets out's own error (its weights' roundings) and the rest of its
      # rounding; dS is rounded once
      tds = (HB + rp) * ds.abs() + p * ((e.abs() * (to - (HB - HB * HB) * o.abs())).sum(-1, keepdim=True) +
                                        (v.shape[2] * HF + rp) * (e.abs() @ c.abs().t()))
      res["dv"][0][k0:k0 + lk, h // g] += p.t() @ e
      res["dv"][1][k0:k0 + lk, h // g] += (HB + rp) * (p.t() @ e.abs())
      res["dq"][0][q0:q0 + lq, h] += ds @ b * scale
      res["dq"][1][q0:q0 + lq, h] += tds @ b.abs() * scale
      res["dk"][0][k0:k0 + lk, h // g] += ds.t() @ a * scale
      res["dk"][1][k0:k0 + lk, h // g] += tds.t() @ a.abs() * scale
  if dout is not None:
    for name in ("dq", "dk", "dv"):
      want, tol = res[name]
      # the result's own rounding, and the fp32 sums behind the bf16 products
      res[name] = (want, tol * (1 + 2.0 ** -6) + HB * want.abs() + 1e-30)
  return res


def run_attention(K, Fn, q_lengths, k_lengths, heads, kv_heads, d, dv, causal, grad, seed=0, q_starts=None, k_starts=None,
                  scale=None, spread=1.0, rows=None):
  gen = torch.Generator().manual_seed(seed)
  plan = K.AttentionPlan(q_lengths, k_lengths, heads=heads, kv_heads=kv_heads, causal=causal, q_starts=q_starts,
                         k_starts=k_starts)
  kl = list(q_lengths) if k_lengths is None else list(k_lengths)
  q0 = list(q_starts) if q_starts else [sum(q_lengths[:i]) for i in range(len(q_lengths))]
  k0 = list(k_starts) if k_starts else [sum(kl[:i]) for i in range(len(kl))]
  nq, nk = rows or (plan.q_rows, plan.k_rows)
  q = (spread * normal(gen, (nq, heads, d))).cuda().requires_grad_(grad)
  k = (spread * normal(gen, (nk, kv_heads, d))).cuda().requires_grad_(grad)
  v = normal(gen, (nk, kv_heads, dv)).cuda().requires_grad_(grad)
  dout = normal(gen, (nq, heads, dv)).cuda() if grad else None
  out = Fn.packed_attention(q, k, v, plan, scale)
  got = {"out": out}
  if grad:
    got["dq"], got["dk"], got["dv"] = torch.autograd.grad(out, (q, k, v), dout)
  want = exact_attention(q.detach(), k.detach(), v.detach(), dout, list(zip(q0, q_lengths, k0, kl)), heads, kv_heads,
                         causal, 1.0 / math.sqrt(d) if scale is None else scale)
  for name, (value, tol) in want.items():
    within(got[name], value, tol, name)
  return got, (q, k, v, dout, plan)


ATTENTION = [
    # q_lengths, k_lengths, heads, kv_heads, D, Dv, causal
    ([1], None, 1, 1, 8, 8, False),
    ([1], [1], 4, 1, 64, 64, True),
    ([1], [2], 40, 1, 128, 128, True),
    ([16] * 9, None, 3, 3, 64, 64, False),
    ([32], [33], 1, 1, 32, 32, False),
    ([33], [32], 1, 1, 32, 32, True),
    ([64, 1, 0, 63, 65], None, 4, 2, 64, 64, True),
    ([127, 129, 128], None, 2, 1, 128, 128, True),
    ([127, 129, 128], None, 2, 1, 128, 128, False),
    ([100], [40], 3, 1, 96, 64, True),              # rows in front of the keys see nothing
    ([40], [300], 6, 2, 64, 128, True),
    ([5, 0, 7, 9], [0, 6, 200, 1], 5, 5, 40, 72, False),
    ([300, 257], None, 5, 1, 8, 120, True),
    ([513], None, 2, 2, 104, 104, False),
    ([1000], [1100], 1, 1, 128, 128, True),
    ([7], [1900], 3, 1, 64, 64, True),
    # small sequences beside large ones: in the large ones' launches, and (many) in their own
    ([3, 200, 1, 0, 17, 32, 8], None, 2, 2, 64, 64, True),
    ([1, 4, 150, 2], [30, 0, 150, 7], 4, 1, 48, 64, True),
    ([7] * 90 + [140], None, 3, 3, 32, 40, False),
    # key and value widths in every pair of the kernels' widths of 32, 64, 96 and 128
    ([130, 17], None, 2, 1, 128, 32, True),
    ([130, 17], None, 2, 1, 16, 128, True),
    ([200], [150], 2, 2, 128, 96, False),
    ([150], [200], 4, 1, 96, 128, True),
    ([150, 3], None, 2, 1, 32, 64, True),
    ([150, 3], None, 2, 1, 64, 32, False),
    ([150, 65], None, 2, 1, 24, 80, True),
    ([150, 65], None, 2, 1, 88, 24, True),
    ([133, 20], None, 2, 1, 48, 96, True),
    ([133, 20], None, 2, 1, 120, 48, False),
    ([133, 20], None, 2, 1, 96, 88, True),
]


@pytest.mark.parametrize("case", ATTENTION, ids=[str(i) for i in range(len(ATTENTION))])
def test_packed_attention(K, Fn, case):
  run_attention(K, Fn, *case, grad=True, seed=len(case[0]) + case[4])


NEW_TOKENS = [
    # k_lengths, heads, kv_heads, D, Dv, capacity
    ([1, 513, 0, 4097], 8, 2, 128, 128, 5000),
    ([129, 128], 32, 1, 64, 64, 129),
    ([20000], 8, 8, 128, 128, 20000),
    ([9001, 3], 12, 4, 96, 32, 9001),
    ([70000], 1, 1, 32, 32, 70000),
    ([5, 2000, 0, 128, 40, 129, 1], 8, 2, 64, 96, 2000),
    ([3] * 299 + [900], 4, 1, 64, 64, 1000),
    ([131072], 2, 2, 128, 8, 131072),               # hundreds of parts for one row
    ([60000, 9], 9, 3, 16, 40, 60001),
    ([3001], 66, 2, 64, 64, 3001),                  # 33 shared heads: more than one wave's rows
]


@pytest.mark.parametrize("case", NEW_TOKENS, ids=[str(i) for i in range(len(NEW_TOKENS))])
def test_new_tokens_against_a_cache(K, Fn, case):
  k, heads, kv_heads, d, dv, capacity = case
  n = len(k)
  run_attention(K, Fn, [1] * n, k, heads, kv_heads, d, dv, True, False, k_starts=[i * capacity for i in range(n)],
                rows=(n, n * capacity))


def test_split_over_keys_with_many_rows(K, Fn):
  """Few tiles of 128 rows against many keys: partial results joined; with gradients."""
  run_attention(K, Fn, [70], [5000], 2, 1, 64, 64, True, True)
  run_attention(K, Fn, [300, 3], [3000, 2000], 1, 1, 128, 96, False, True)
  run_attention(K, Fn, [16], [40000], 4, 1, 72, 40, True, True)       # tens of parts a tile


@pytest.mark.parametrize("spread", [0.0, 8.0])
def test_flat_and_sharp_scores(K, Fn, spread):
  """All scores equal, and scores so far apart that the reference exponent is raised again and again."""
  run_attention(K, Fn, [150], [400], 2, 2, 64, 64, False, spread == 0.0, spread=spread)


def test_scale(K, Fn):
  run_attention(K, Fn, [90], None, 2, 1, 32, 32, True, True, scale=0.7)
  run_attention(K, Fn, [90], None, 2, 1, 32, 32, True, True, scale=1e-3)


def test_rising_scores_raise_the_reference(K, Fn):
  """Every tile's maximum passes the last one's by far: the accumulators are rescaled in every tile."""
  d, n = 64, 512
  k = torch.zeros(n, 1, d)
  k[:, 0, 0] = torch.arange(n) / 4.0
  q = torch.zeros(130, 1, d)
  q[:, 0, 0] = torch.linspace(-8, 8, 130)
  v = normal(torch.Generator().manual_seed(1), (n, 1, d))
  q, k = q.bfloat16(), k.bfloat16()
  plan = K.AttentionPlan([130], [n], heads=1)
  got = Fn.packed_attention(q.cuda(), k.cuda(), v.cuda(), plan, 1.0)
  want = exact_attention(q, k, v, None, [(0, 130, 0, n)], 1, 1, False, 1.0)["out"]
  within(got, want[0], want[1], "out")


def test_padded_batch_and_rows_of_nobody(K, Fn):
  """Starts with room between the sequences, filled with NaN: nothing of it is read into a result; rows of nobody
  give zeros and get zero gradients, and keep what a given output holds."""
  cap, lens, heads = 96, [50, 0, 96, 7], 2
  starts = [i * cap for i in range(4)]
  plan = K.AttentionPlan(lens, heads=heads, causal=True, q_starts=starts, k_starts=starts)
  gen = torch.Generator().manual_seed(3)
  rows = 4 * cap + 5
  mine = torch.zeros(rows, dtype=torch.bool)
  for s, n in zip(starts, lens):
    mine[s:s + n] = True
  data = []
  for _ in range(4):
    x = normal(gen, (rows, heads, 64))
    x[~mine] = float("nan")
    data.append(x.cuda())
  q, k, v, dout = data
  for x in (q, k, v):
    x.requires_grad_(True)
  out = Fn.packed_attention(q, k, v, plan)
  got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(out, (q, k, v), dout)), out=out)
  clean = [x.detach().nan_to_num(0.0) for x in data]
  want = exact_attention(*clean, list(zip(starts, lens, starts, lens)), heads, heads, True, 0.125)
  for name, (value, tol) in want.items():
    within(got[name], value, tol, name)
    assert torch.equal(got[name][~mine], torch.zeros_like(got[name][~mine]))
  kept = torch.full((rows, heads, 64), 3.0, dtype=torch.bfloat16, device="cuda")
  K.packed_attention_fwd(q.detach(), k.detach(), v.detach(), plan, out=kept)
  assert torch.equal(kept[~mine], torch.full_like(kept[~mine], 3.0))
  within(kept[mine], want["out"][0][mine], want["out"][1][mine], "kept")


def test_strided_and_merged_inputs(K, Fn):
  """q, k, v as views of one projection, broadcast heads, odd strides (copied), gradients of the views."""
  gen = torch.Generator().manual_seed(4)
  lens, seqs = [70, 33], [(0, 70, 0, 70), (70, 33, 70, 33)]
  plan = K.AttentionPlan(lens, heads=4, kv_heads=2, causal=True)
  merged = normal(gen, (103, 8, 64)).cuda().requires_grad_(True)
  q, k, v = merged[:, :4], merged[:, 4:6], merged[:, 6:]
  dout = normal(gen, (103, 4, 64)).cuda()
  out = Fn.packed_attention(q, k, v, plan)
  (dm,) = torch.autograd.grad(out, (merged,), dout)
  want = exact_attention(q.detach(), k.detach(), v.detach(), dout, seqs, 4, 2, True, 0.125)
  within(out, *want["out"], "out")
  for name, got in (("dq", dm[:, :4]), ("dk", dm[:, 4:6]), ("dv", dm[:, 6:])):
    within(got, *want[name], name)
  # one key head shown to all by a stride of zero, odd row strides, a transposed width
  one = normal(gen, (103, 1, 64)).cuda()
  odd = normal(gen, (103, 4, 67)).cuda()[..., 1:65]
  turned = normal(gen, (103, 64, 2)).cuda().transpose(1, 2)
  out = Fn.packed_attention(odd, one.expand(103, 2, 64), turned, plan)
  want = exact_attention(odd, one.expand(103, 2, 64), turned, None, seqs, 4, 2, True, 0.125)
  within(out, *want["out"], "strided")


def test_no_keys_at_all(K, Fn):
  plan = K.AttentionPlan([3, 2], [0, 0], heads=2)
  q = torch.ones((5, 2, 16), dtype=torch.bfloat16, device="cuda", requires_grad=True)
  k = torch.ones((0, 2, 16), dtype=torch.bfloat16, device="cuda", requires_grad=True)
  out = Fn.packed_attention(q, k, k, plan)
  assert torch.equal(out, torch.zeros_like(out))
  dq, dk = torch.autograd.grad(out, (q, k), torch.ones_like(out))
  assert torch.equal(dq, torch.zeros_like(dq)) and dk.shape == k.shape
  plan = K.AttentionPlan([0], [4], heads=2)
  q0 = torch.ones((0, 2, 16), dtype=torch.bfloat16, device="cuda", requires_grad=True)
  k4 = torch.ones((4, 2, 16), dtype=torch.bfloat16, device="cuda", requires_grad=True)
  out = Fn.packed_attention(q0, k4, k4, plan)
  dk = torch.autograd.grad(out, (k4,), torch.ones_like(out))[0]
  assert out.shape == (0, 2, 16) and torch.equal(dk, torch.zeros_like(dk))


def test_statistics_of_rows(K):
  gen = torch.Generator().manual_seed(6)
  q, k = normal(gen, (40, 1, 32)), normal(gen, (20, 1, 32))
  plan = K.AttentionPlan([40], [20], causal=True)
  out, (lse, _) = K.packed_attention_fwd(q.cuda(), k.cuda(), k.cuda(), plan)
  s = q[:, 0].double() @ k[:, 0].double().t() / math.sqrt(32)
  s = s.masked_fill(torch.arange(20)[None] > torch.arange(40)[:, None] - 20, -math.inf)
  want = torch.logsumexp(s, -1)
  assert (lse[:20, 0] == -math.inf).all() and (out[:20] == 0).all()
  assert ((lse[20:, 0].cpu() - want[20:]).abs() < 1e-5).all()
  assert K.packed_attention_fwd(q.cuda(), k.cuda(), k.cuda(), plan, want_grad=False)[1] is None


def test_infinite_and_missing_values_stay_in_their_rows(K, Fn):
  """A NaN in a query, and an infinite one, reach that row only; NaN in a key's row reach every row that sees it."""
  gen = torch.Generator().manual_seed(7)
  q, k, v = (normal(gen, (200, 1, 64)).cuda() for _ in range(3))
  plan = K.AttentionPlan([200])
  clean = Fn.packed_attention(q, k, v, plan)
  q[17, 0, 3] = float("nan")
  q[90, 0, 5] = float("inf")
  got = Fn.packed_attention(q, k, v, plan)
  rest = torch.ones(200, dtype=torch.bool)
  rest[[17, 90]] = False
  assert torch.equal(got[rest], clean[rest])
  assert got[17].isnan().all() and got[90].isnan().all()
  k[3, 0, 0] = float("nan")
  assert Fn.packed_attention(q, k, v, plan).isnan().all()


MASKED_PLACES = [
    # lengths, heads, kv_heads, D, the poisoned token of the first sequence
    ([40], 2, 2, 64, 25), ([20], 1, 1, 128, 7), ([9, 9], 3, 1, 32, 8), ([300], 2, 1, 64, 130), ([700], 1, 1, 128, 699),
    ([129], 4, 1, 96, 0), ([2100], 1, 1, 64, 2049), ([64, 64], 2, 2, 32, 63),
]


@pytest.mark.parametrize("poison", [float("nan"), float("inf")])
@pytest.mark.parametrize("case", MASKED_PLACES, ids=[str(i) for i in range(len(MASKED_PLACES))])
def test_values_that_are_not_finite_in_masked_places(K, Fn, case, poison):
  """A token whose key and value (query and incoming gradient) are not finite, causal: every result that does not see it
  is the clean one to the bit, every one that does is not finite."""
  lens, heads, kv_heads, d, at = case
  gen = torch.Generator().manual_seed(at)
  n = sum(lens)
  plan = K.AttentionPlan(lens, heads=heads, kv_heads=kv_heads, causal=True)
  q, k, v = (normal(gen, (n, h, d)).cuda() for h in (heads, kv_heads, kv_heads))
  dout = normal(gen, (n, heads, d)).cuda()

  def run(q, k, v, dout):
    out, saved = K.packed_attention_fwd(q, k, v, plan)
    return (out,) + K.packed_attention_bwd(q, k, v, plan, out, saved, dout)
  clean = run(q, k, v, dout)
  see = torch.zeros(n, dtype=torch.bool)             # rows that see the token's key
  see[at:lens[0]] = True
  seen = torch.zeros(n, dtype=torch.bool)            # keys that the token's row sees
  seen[:at + 1] = True
  for which in ("k", "v"):
    kk, vv = k.clone(), v.clone()
    (kk if which == "k" else vv)[at, :, 3] = poison
    got = run(q, kk, vv, dout)
    for x, y in zip(got[:2], clean[:2]):             # out, dq
      assert torch.equal(x[~see], y[~see])
      if which == "v" or poison != poison:           # (an infinite key may give a weight of 0)
        assert (~torch.isfinite(x[see].float())).any(-1).all()
    for x, y in zip(got[2:], clean[2:]):             # dk, dv of keys behind: no row that sees the token sees more
      behind = torch.zeros(n, dtype=torch.bool)
      behind[lens[0]:] = True
      assert torch.equal(x[behind], y[behind])
  for which in ("q", "dout"):
    qq, dd = q.clone(), dout.clone()
    (qq if which == "q" else dd)[at, :, 3] = poison
    got = run(qq, k, v, dd)
    own = torch.zeros(n, dtype=torch.bool)
    own[at] = True
    assert torch.equal(got[1][~own], clean[1][~own])
    for x, y in zip(got[2:], clean[2:]):             # dk, dv of the keys that the row does not see
      assert torch.equal(x[~seen], y[~seen])
      if poison != poison:
        assert (~torch.isfinite(x[seen].float())).any(-1).all()


def test_new_token_with_values_that_are_not_finite_behind_it(K, Fn):
  """Chunk of 6 new tokens against a cache, the last ones not finite: the first ones see nothing of them."""
  gen = torch.Generator().manual_seed(2)
  q, k, v = normal(gen, (6, 4, 64)).cuda(), normal(gen, (1000, 1, 64)).cuda(), normal(gen, (1000, 1, 64)).cuda()
  plan = K.AttentionPlan([6], [1000], heads=4, kv_heads=1, causal=True)
  clean = Fn.packed_attention(q, k, v, plan)
  k[998:] = float("nan")
  v[997:] = float("inf")
  got = Fn.packed_attention(q, k, v, plan)
  assert torch.equal(got[:3], clean[:3]) and not torch.isfinite(got[3:].float()).any(-1).any()


def test_rows_beyond_32_bits(K, Fn):
  """Keys, values and tokens whose offsets pass 2^31 elements: the results of the same rows at the front, to the bit."""
  far, lens = 17_000_000, [300, 70, 1]                     # x 128 entries: 2.2e9
  gen = torch.Generator().manual_seed(12)
  n = sum(lens)
  q, dout = (normal(gen, (n, 2, 128)).cuda() for _ in range(2))
  near = [normal(gen, (n, 1, 128)).cuda() for _ in range(2)]
  starts = [0, far - 80, far - 1]
  big = [torch.empty((far, 1, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
  at = 0
  for s, m in zip(starts, lens):
    for b, x in zip(big, near):
      b[s:s + m] = x[at:at + m]
    at += m
  plans = [K.AttentionPlan(lens, heads=2, kv_heads=1, causal=True, k_starts=x, device="cuda") for x in (None, starts)]
  results = []
  for plan, (k, v) in zip(plans, (near, big)):
    out, saved = K.packed_attention_fwd(q, k, v, plan)
    dq, dk, dv = K.packed_attention_bwd(q, k, v, plan, out, saved, dout)
    if k is big[0]:
      dk, dv = (torch.cat([x[s:s + m] for s, m in zip(starts, lens)]) for x in (dk, dv))
    results.append((out, dq, dk, dv))
  for a, b in zip(*results):
    assert torch.equal(a, b)
  # one new token whose cache lies behind 2^31, and a rotation of far rows
  new = K.AttentionPlan([1, 1, 1], lens, heads=2, kv_heads=1, causal=True)
  there = K.AttentionPlan([1, 1, 1], lens, heads=2, kv_heads=1, causal=True, k_starts=starts)
  assert torch.equal(K.packed_attention_fwd(q[:3], *near, new, want_grad=False)[0],
                     K.packed_attention_fwd(q[:3], *big, there, want_grad=False)[0])
  table, pos = K.RotaryTable(128), torch.arange(100, dtype=torch.int32, device="cuda")
  rows = big[0][::170_000]
  rows.copy_(q[:100, :1])
  assert torch.equal(K.rotary(rows, pos, table), K.rotary(q[:100, :1].contiguous(), pos, table))


def test_same_result_every_time(K, Fn):
  """No atomics: two runs agree to the bit, alone and with another stream's call in between."""
  gen = torch.Generator().manual_seed(8)
  q, k, v = (normal(gen, (700, h, 64)).cuda().requires_grad_(True) for h in (4, 2, 2))
  dout = normal(gen, (700, 4, 64)).cuda()
  plan = K.AttentionPlan([300, 400], heads=4, kv_heads=2, causal=True)

  def once():
    out = Fn.packed_attention(q, k, v, plan)
    return (out.detach(),) + torch.autograd.grad(out, (q, k, v), dout)
  first = once()
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    other = once()
  second = once()
  torch.cuda.synchronize()
  for a, b, c in zip(first, second, other):
    assert torch.equal(a, b) and torch.equal(a, c)


def test_gradients_against_differences(K, Fn):
  """d/de of sum(dout * out) along a random direction, taken from the kernels' own outputs at q, k, v +- e dir."""
  gen = torch.Generator().manual_seed(9)
  lens, heads, kv_heads, d = [60, 45], 4, 2, 64
  plan = K.AttentionPlan(lens, heads=heads, kv_heads=kv_heads, causal=True)
  n = sum(lens)
  q, k, v = (normal(gen, (n, h, d)).cuda().requires_grad_(True) for h in (heads, kv_heads, kv_heads))
  dout = normal(gen, (n, heads, d)).cuda()
  grads = torch.autograd.grad(Fn.packed_attention(q, k, v, plan), (q, k, v), dout)
  for i, x in enumerate((q, k, v)):
    # along the gradient itself: the derivative is large against the rounding of the outputs
    step = 0.5 * grads[i].float() / grads[i].float().abs().max()
    up, down = ((x.detach().float() + s * step).bfloat16() for s in (1, -1))
    args = [[y.detach() for y in (q, k, v)] for _ in range(2)]
    args[0][i], args[1][i] = up, down
    a, b = (Fn.packed_attention(*xs, plan).double() for xs in args)
    change = float((dout.double() * (a - b)).sum())
    want = float((grads[i].double() * (up.double() - down.double())).sum())
    # third derivative: a step of at most 1/2 in values of size 1, softmax slopes of size 1: a few percent
    assert abs(change - want) <= 0.05 * abs(want), (i, change, want)


def test_attention_refusals(K, Fn):
  plan = K.AttentionPlan([4], heads=2, kv_heads=1)
  z = lambda *s, **kw: torch.zeros(s, dtype=kw.get("dtype", torch.bfloat16), device="cuda")
  good = dict(q=z(4, 2, 16), k=z(4, 1, 16), v=z(4, 1, 24), plan=plan)
  assert Fn.packed_attention(**good).shape == (4, 2, 24)
  for bad in (dict(q=z(4, 2, 16, dtype=torch.float32)), dict(k=z(4, 1, 16, dtype=torch.half)), dict(q=z(4, 1, 16)),
              dict(k=z(4, 2, 16)), dict(k=z(4, 1, 24)), dict(v=z(5, 1, 24)), dict(q=z(3, 2, 16)),
              dict(k=z(3, 1, 16), v=z(3, 1, 16)), dict(q=z(4, 2, 12), k=z(4, 1, 12)), dict(v=z(4, 1, 136)),
              dict(q=z(4, 32)), dict(plan=None), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=1e300), dict(scale=1e-60),
              dict(plan=K.AttentionPlan([4], heads=2, kv_heads=1, device="cpu")), dict(v=z(4, 1, 24).cpu())):
    with pytest.raises(ValueError):
      Fn.packed_attention(**dict(good, **bad))
  with pytest.raises(ValueError):
    K.packed_attention_fwd(out=z(4, 2, 16), **good)
  out, saved = K.packed_attention_fwd(**good)
  with pytest.raises(ValueError):
    K.packed_attention_bwd(good["q"], good["k"], good["v"], plan, out, saved, z(4, 2, 16))
  with pytest.raises(ValueError):
    K.packed_attention_bwd(good["q"], good["k"], good["v"], plan, out, None, out)
  q = z(4, 2, 16).requires_grad_(True)                # no second derivative: refused, not wrong
  out = Fn.packed_attention(q, good["k"], good["v"], plan)
  (dq,) = torch.autograd.grad(out.float().sum(), (q,), create_graph=True)
  with pytest.raises(RuntimeError):
    dq.float().sum().backward()


@pytest.mark.parametrize("seed", range(6))
def test_drawn_sequences(K, Fn, seed):
  rng = random.Random(seed)
  n = rng.randint(1, 6)
  q = [rng.choice((0, 1, 2, 31, 32, 33, 64, rng.randint(1, 400))) for _ in range(n)]
  k = None if rng.random() < 0.4 else [rng.choice((0, 1, 63, 64, 65, rng.randint(1, 600))) for _ in range(n)]
  kv_heads = rng.randint(1, 3)
  heads = kv_heads * rng.randint(1, 4)
  if not any(q):
    q[0] = 1
  run_attention(K, Fn, q, k, heads, kv_heads, 8 * rng.randint(1, 16), 8 * rng.randint(1, 16), rng.random() < 0.5, True,
                seed=seed)


# ------------------------------------------------------------------------------------------------
# together
# ------------------------------------------------------------------------------------------------
def test_block_of_the_three(K, Fn):
  """Projection rows -> norm + rotation -> attention, with gradients back to the projection and the gains, against
  the chain in 64 bits; relative error of whole tensors (each stage rounds to bf16: three roundings of half a step
  2^-8 each, uncorrelated over the sums)."""
  gen = torch.Generator().manual_seed(11)
  lens, heads, kv_heads, d = [64, 100, 1, 37], 4, 2, 64
  n = sum(lens)
  merged = normal(gen, (n, heads + 2 * kv_heads, d)).cuda().requires_grad_(True)
  qg, kg = ((1 + 0.2 * normal(gen, (d,), torch.float32)).cuda().requires_grad_(True) for _ in range(2))
  pos = torch.cat([torch.arange(x) for x in lens]).int().cuda()
  table = K.RotaryTable(d)
  plan = K.AttentionPlan(lens, heads=heads, kv_heads=kv_heads, causal=True)
  q, k = Fn.qk_norm_rotary(merged[:, :heads], merged[:, heads:heads + kv_heads], qg, kg, pos, table)
  out = Fn.packed_attention(q, k, merged[:, heads + kv_heads:], plan)
  dout = normal(gen, out.shape).cuda()
  got = (out,) + torch.autograd.grad(out, (merged, qg, kg), dout)
  m = merged.detach().double().cpu().requires_grad_(True)
  a, b = (x.detach().double().cpu().requires_grad_(True) for x in (qg, kg))
  f = table.freq.cpu() * 2 * math.pi
  angle = (pos.cpu().double()[:, None] * f)[:, None]
  cos, sin = torch.cos(angle), torch.sin(angle)

  def turn(x):
    y, z = x[..., :d // 2], x[..., d // 2:]
    return torch.cat((y * cos - z * sin, y * sin + z * cos), -1)
  qq = turn(exact_norm(m[:, :heads], a, 1e-6))
  kk = turn(exact_norm(m[:, heads:heads + kv_heads], b, 1e-6))
  vv = m[:, heads + kv_heads:]
  outs, at = [], 0
  for x in lens:
    part = []
    for h in range(heads):
      s = qq[at:at + x, h] @ kk[at:at + x, h // 2].t() / 8.0
      s = s.masked_fill(torch.ones(x, x, dtype=torch.bool).triu(1), -math.inf)
      part.append(torch.softmax(s, -1) @ vv[at:at + x, h // 2])
    outs.append(torch.stack(part, 1))
    at += x
  o = torch.cat(outs)
  want = (o,) + torch.autograd.grad(o, (m, a, b), dout.double().cpu())
  for name, x, y in zip(("out", "dmerged", "dq_gain", "dk_gain"), got, want):
    x, y = x.detach().double().cpu(), y.detach()
    assert float((x - y).norm() / y.norm()) <= 3 * HB, name


def test_captured_and_replayed(K, Fn):
  """Forward and backward of the three in one graph (direct calls: no autograd inside the capture), replayed with new
  inputs and eager work in between."""
  gen = torch.Generator().manual_seed(12)
  lens, heads, kv_heads, d = [1, 130, 70], 4, 1, 64
  n = sum(lens)
  plan = K.AttentionPlan(lens, [1, 900, 70], heads=heads, kv_heads=kv_heads, causal=True)
  table = K.RotaryTable(d)
  pos = torch.arange(n, dtype=torch.int32, device="cuda")
  gain = torch.ones(d, device="cuda")
  q, k = normal(gen, (n, heads, d)).cuda(), normal(gen, (n, kv_heads, d)).cuda()
  cache_k, cache_v = (normal(gen, (971, kv_heads, d)).cuda() for _ in range(2))
  dout = normal(gen, (n, heads, d)).cuda()

  def step():
    a, b = K.qk_norm_rotary(q, k, gain, gain, pos, table)
    out, saved = K.packed_attention_fwd(a, cache_k, cache_v, plan)
    grads = K.packed_attention_bwd(a, cache_k, cache_v, plan, out, saved, dout)
    back = K.qk_norm_rotary_bwd(q, k, gain, gain, pos, table, grads[0], b)
    return (out, K.rotary(b, pos, table)) + grads + back
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    step()
  torch.cuda.current_stream().wait_stream(side)
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    held = step()
  for i in range(4):
    q.copy_(normal(gen, q.shape))
    cache_k.copy_(normal(gen, cache_k.shape))
    want = [x.clone() for x in step()]
    graph.replay()
    torch.cuda.synchronize()
    for x, y in zip(held, want):
      assert torch.equal(x, y), i


# ------------------------------------------------------------------------------------------------
# entries behind the turned part
# ------------------------------------------------------------------------------------------------
# D, rot: the last turned pairs and the first copied entries share a load of 8, 4 (twice) or 2 pairs, or none
BEHIND = [(32, 20), (72, 36), (24, 14), (20, 14), (18, 10), (64, 32)]


def same_bits(a, b):
  word = {2: torch.int16, 4: torch.int32}[a.element_size()]
  return torch.equal(a.contiguous().view(word), b.contiguous().view(word))


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d,rot", BEHIND)
def test_entries_behind_the_turned_part_are_copied(K, Fn, d, rot, dtype, layout):
  """To the bit, whatever lies beside them (infinities, NaN, zeros of either sign), and the turned part does not notice."""
  gen = torch.Generator().manual_seed(d)
  table, pos = K.RotaryTable(rot, layout=layout), positions_of(gen, 9, 1, 1000)
  clean = normal(gen, (9, 3, d), dtype).cuda()
  want = K.rotary(clean, pos, table)
  for poison in (float("inf"), float("-inf"), float("nan"), 0.0, -0.0):
    for at in range(rot, min(rot + 8, d)):
      x = clean.clone()
      x[::2, 1:, at] = poison
      for inverse in (False, True):
        y = K.rotary(x, pos, table, inverse=inverse)
        assert same_bits(y[..., rot:], x[..., rot:]), (poison, at)
        if not inverse:
          assert same_bits(y[..., :rot], want[..., :rot]), (poison, at)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d,rot", BEHIND)
def test_norm_beside_copied_entries_that_are_not_finite(K, Fn, d, rot, dtype):
  """An infinite copied entry makes the head's norm infinite: it becomes NaN and the others 0, as the formula has it.  An
  infinite incoming gradient of a copied entry reaches its own row and its own gain, no other."""
  gen = torch.Generator().manual_seed(d + 1)
  table, pos = K.RotaryTable(rot, layout="interleaved"), positions_of(gen, 9, 1, 1000)
  q, k = normal(gen, (9, 3, d), dtype).cuda(), normal(gen, (9, 1, d), dtype).cuda()
  gain = torch.ones(d, device="cuda")
  dq, dk = normal(gen, q.shape, dtype).cuda(), normal(gen, k.shape, dtype).cuda()
  clean = K.qk_norm_rotary(q, k, gain, gain, pos, table)
  grads = K.qk_norm_rotary_bwd(q, k, gain, gain, pos, table, dq, dk)
  for at in range(rot, min(rot + 8, d)):
    x = q.clone()
    x[4, 1, at] = float("inf")
    y = K.qk_norm_rotary(x, k, gain, gain, pos, table)[0]
    want = clean[0].clone()
    want[4, 1] = 0.0
    assert y[4, 1, at].isnan()
    y[4, 1, at] = 0.0
    assert torch.equal(y, want), at
    dy = dq.clone()
    dy[4, 1, at] = float("inf")
    got = K.qk_norm_rotary_bwd(q, k, gain, gain, pos, table, dy, dk)
    rest = torch.arange(d, device="cuda") != at
    assert torch.equal(got[2][rest], grads[2][rest]) and not torch.isfinite(got[2][at]), at
    got[0][4, 1], grads[0][4, 1] = 0.0, 0.0
    assert torch.equal(got[0], grads[0]) and torch.equal(got[1], grads[1]) and torch.equal(got[3], grads[3])


def test_plan_and_table_dropped_while_another_stream_reads_them(K, Fn):
  """Their memory is not given to other tensors before that stream is done (nothing is written to those here), and the
  results are the ones of a plan and a table that live on."""
  gen = torch.Generator().manual_seed(13)
  lens = [1 + (i * 37) % 300 for i in range(60)]
  n = sum(lens)
  q, pos = normal(gen, (n, 2, 64)).cuda(), torch.arange(n, dtype=torch.int32, device="cuda")

  def make():
    return K.RotaryTable(64), K.AttentionPlan(lens, heads=2, causal=True)

  def call(table, plan):
    return Fn.packed_attention(Fn.rotary(q, pos, table), q, q, plan)
  table, plan = make()
  want = call(table, plan)
  busy = torch.randn((4096, 4096), device="cuda").bfloat16()
  torch.matmul(busy, busy)
  side = torch.cuda.Stream()
  torch.cuda.synchronize()
  del table, plan
  table, plan = make()
  places = {table.freq.data_ptr(): table.freq.numel() * 8, plan.data.data_ptr(): plan.data.numel() * 4}
  with torch.cuda.stream(side):
    for _ in range(1500):            # a tenth of a second and more in front of the call
      torch.matmul(busy, busy)
    got = call(table, plan)
    done = torch.cuda.Event()
    done.record()
  del table, plan
  others = [torch.empty(size, dtype=torch.uint8, device="cuda") for size in places.values() for _ in range(8)]
  assert not done.query(), "the other stream was done before the test looked"
  assert not {x.data_ptr() for x in others} & set(places)
  torch.cuda.synchronize()
  assert torch.equal(got, want)


def test_an_output_that_is_an_input_is_refused(K):
  """Rows are read until the last work item is done, so none of them may be written before."""
  gen = torch.Generator().manual_seed(14)
  plan = K.AttentionPlan([300], heads=2)
  q, k, v = (normal(gen, (300, 2, 64)).cuda() for _ in range(3))
  want = K.packed_attention_fwd(q, k, v, plan)[0]
  for out in (q, k, v):
    with pytest.raises(ValueError, match="share memory"):
      K.packed_attention_fwd(q, k, v, plan, out=out)
  # neighbours in one buffer are not each other's memory; a single token's row holds q, k, v and the output
  buffer = torch.zeros((2, 300, 2, 64), dtype=torch.bfloat16, device="cuda")
  buffer[0] = q
  assert torch.equal(K.packed_attention_fwd(buffer[0], k, v, plan, out=buffer[1])[0], want)
  row = normal(gen, (1, 8, 64)).cuda()
  one = K.AttentionPlan([1], heads=2)
  got = K.packed_attention_fwd(row[:, :2], row[:, 2:4], row[:, 4:6], one, out=row[:, 6:])[0]
  assert torch.equal(got, row[:, 4:6]) and torch.equal(row[:, 6:], row[:, 4:6])


# ------------------------------------------------------------------------------------------------
# split items: nothing lost, nothing twice
# ------------------------------------------------------------------------------------------------
# The entry by entry bounds above are worst cases: where a row sees many keys whose values cancel they are as large as the
# result, and a lost part hides in them.  So (a) whole tensors by their norm: inputs are independent and of zero mean,
# so the errors of the rounded weights add up like the results themselves, HB / sqrt(3) of the norm, and the result's own
# rounding is at most HB of it: 2 HB in all for out and dv (1.6 counted); dq and dk also carry delta's error, HB / sqrt(3)
# again, and dP's: 3 HB (2.2 counted).  One lost part of n is 1 / sqrt(n) of the norm, 16 HB for 256 parts.
def run_norms(K, Fn, *case, grad, **kw):
  got, (q, k, v, dout, plan) = run_attention(K, Fn, *case, grad=grad, **kw)
  q_lengths, k_lengths, heads, kv_heads, d, _, causal = case
  kl = q_lengths if k_lengths is None else k_lengths
  k0 = kw.get("k_starts") or [sum(kl[:i]) for i in range(len(kl))]
  seqs = list(zip([sum(q_lengths[:i]) for i in range(len(q_lengths))], q_lengths, k0, kl))
  want = exact_attention(q.detach(), k.detach(), v.detach(), dout, seqs, heads, kv_heads, causal, 1.0 / math.sqrt(d))
  for name, (value, _) in want.items():
    error = float((got[name].detach().double().cpu() - value).norm() / value.norm())
    assert error <= (2 if name in ("out", "dv") else 3) * HB, (name, error)
  return plan


@pytest.mark.parametrize("case", NEW_TOKENS, ids=[str(i) for i in range(len(NEW_TOKENS))])
def test_norm_of_new_tokens_against_a_cache(K, Fn, case):
  k, heads, kv_heads, d, dv, capacity = case
  n = len(k)
  run_norms(K, Fn, [1] * n, k, heads, kv_heads, d, dv, True, grad=False, k_starts=[i * capacity for i in range(n)],
            rows=(n, n * capacity))


SPLIT = [
    # q_lengths, k_lengths, heads, kv_heads, D, Dv, causal, what is split
    ([70], [5000], 2, 1, 64, 64, True, "parts dq_parts"),
    ([300, 3], [3000, 2000], 1, 1, 128, 96, False, "parts dq_parts"),
    ([16], [40000], 4, 1, 72, 40, True, "parts dq_parts"),
    ([40000], [16], 4, 1, 72, 40, False, "dkv_parts"),
    ([9000], [200], 2, 2, 128, 128, False, "dkv_parts"),
    ([4000], None, 2, 1, 64, 32, True, "parts dq_parts dkv_parts"),
]


@pytest.mark.parametrize("case", SPLIT, ids=[str(i) for i in range(len(SPLIT))])
def test_norm_of_split_items(K, Fn, case):
  plan = run_norms(K, Fn, *case[:7], grad=True)
  for name in case[7].split():
    assert getattr(plan.info, name) > 0, name


# (b) inputs that mark the parts, and only terms of one sign in every sum: the bounds are then 2 HB or so of the result, and
# a part that is lost or taken twice is a whole column (of at most a few blocks of 512)
def marks(n, width):
  x = torch.zeros(n, 1, width)
  x[torch.arange(n), 0, (torch.arange(n) // 512) % width] = 1.0
  return x


@pytest.mark.parametrize("n,rows,heads,kv_heads,d,dv,causal", [
    (131072, 1, 2, 1, 128, 128, True), (70000, 1, 1, 1, 128, 64, True), (40000, 16, 4, 1, 80, 40, True),
    (20000, 150, 2, 1, 64, 64, False), (9001, 1, 12, 4, 24, 24, True), (6000, 300, 1, 1, 128, 128, True)])
def test_every_part_of_the_keys_counts_once(K, Fn, n, rows, heads, kv_heads, d, dv, causal):
  gen = torch.Generator().manual_seed(n)
  plan = K.AttentionPlan([rows], [n], heads=heads, kv_heads=kv_heads, causal=causal)
  assert plan.info.parts > 0 and plan.info.dq_parts > 0
  q = 0.25 * normal(gen, (rows, heads, d), torch.float32)
  k = marks(n, d).expand(n, kv_heads, d)
  sign = 1.0 - 2.0 * ((torch.arange(n) // 512) % 2)
  seqs = [(0, rows, 0, n)]
  for v in (marks(n, dv).expand(n, kv_heads, dv), sign[:, None, None].expand(n, kv_heads, dv)):
    q_, k_, v_ = (x.bfloat16().cuda().requires_grad_(True) for x in (q, k, v))
    dout = normal(gen, (rows, heads, dv)).abs().cuda()
    out = Fn.packed_attention(q_, k_, v_, plan)
    dq, dk, dvalue = torch.autograd.grad(out, (q_, k_, v_), dout)
    want = exact_attention(q_.detach(), k_.detach(), v_.detach(), dout, seqs, heads, kv_heads, causal, 1 / math.sqrt(d))
    for name, got in (("out", out), ("dq", dq), ("dk", dk), ("dv", dvalue)):
      within(got, want[name][0], want[name][1], name)
    if v.min() >= 0:
      assert float((want["out"][1] / want["out"][0].abs().clamp_min(1e-6)).max()) < 3 * HB     # (the bound is tight)
    else:
      assert float((want["dq"][1].norm() / want["dq"][0].norm())) < 5 * HB


@pytest.mark.parametrize("rows,n,heads,kv_heads,d,dv", [(40000, 16, 4, 1, 72, 40), (70000, 40, 1, 1, 128, 128),
                                                      (9000, 200, 2, 2, 64, 24)])
def test_every_part_of_the_rows_counts_once(K, Fn, rows, n, heads, kv_heads, d, dv):
  gen = torch.Generator().manual_seed(n)
  plan = K.AttentionPlan([rows], [n], heads=heads, kv_heads=kv_heads)
  assert plan.info.dkv_parts > 0
  q = marks(rows, d).expand(rows, heads, d).bfloat16().cuda().requires_grad_(True)
  dout = marks(rows, dv).expand(rows, heads, dv).bfloat16().cuda()
  k = (0.25 * normal(gen, (n, kv_heads, d), torch.float32)).bfloat16().cuda().requires_grad_(True)
  v = (1.0 - 2.0 * (torch.arange(n) % 2))[:, None, None].expand(n, kv_heads, dv).bfloat16().cuda().requires_grad_(True)
  out = Fn.packed_attention(q, k, v, plan)
  dq, dk, dvalue = torch.autograd.grad(out, (q, k, v), dout)
  want = exact_attention(q.detach(), k.detach(), v.detach(), dout, [(0, rows, 0, n)], heads, kv_heads, False,
                         1 / math.sqrt(d))
  for name, got in (("out", out), ("dq", dq), ("dk", dk), ("dv", dvalue)):
    within(got, want[name][0], want[name][1], name)
  for name in ("dk", "dv"):
    assert float(want[name][1].norm() / want[name][0].norm()) < 5 * HB, name


@pytest.mark.parametrize("k_lengths,rows,heads,kv_heads,d,dv", [
    ([131072], 1, 2, 2, 128, 8), ([70000], 1, 32, 1, 64, 128),        # groups of threads share a row's parts
    ([4096] * 50, 1, 32, 8, 16, 64),                                  # many joins: a thread a piece of a row
    ([5000], 70, 2, 1, 64, 64), ([3000, 2500], 300, 1, 1, 128, 96)])  # tiles
def test_statistics_of_joined_rows(K, k_lengths, rows, heads, kv_heads, d, dv):
  """lse against the logarithm of the sum in 64 bits: a score is off by D HF sum |q k| scale, the sum is one of at most 512
  + parts fp32 additions in a row, the logarithm and its two products round the result three times."""
  gen = torch.Generator().manual_seed(rows + heads)
  count = len(k_lengths)
  plan = K.AttentionPlan([rows] * count, k_lengths, heads=heads, kv_heads=kv_heads)
  assert plan.info.joins > 0
  q = normal(gen, (rows * count, heads, d))
  k, v = normal(gen, (sum(k_lengths), kv_heads, d)), normal(gen, (sum(k_lengths), kv_heads, dv))
  _, (lse, _) = K.packed_attention_fwd(q.cuda(), k.cuda(), v.cuda(), plan)
  lse = lse.double().cpu()
  at = 0
  for i, n in enumerate(k_lengths):
    for h in range(heads):
      a, b = q[i * rows:(i + 1) * rows, h].double(), k[at:at + n, h * kv_heads // heads].double()
      s = a @ b.t() / math.sqrt(d)
      want = torch.logsumexp(s, -1)
      tol = d * HF * float((a.abs() @ b.abs().t()).max()) / math.sqrt(d) + (512 + plan.info.parts) * HF + 3 * HF * want.abs()
      got = lse[i * rows:(i + 1) * rows, h]
      assert ((got - want).abs() <= tol + 2.0 ** -20).all(), (i, h)
    at += n


# ------------------------------------------------------------------------------------------------
# gain gradients over more blocks of tokens than workgroups
# ------------------------------------------------------------------------------------------------
MANY_TOKENS = [
    # like QK: 16 tokens a block of 256 turned entries, 1032 blocks of them for at most 1024 workgroups, the last one short
    (16507, 1, 1, 256, 256, "half", 1, torch.bfloat16, False, True),
    (16507, 2, 1, 256, 254, "interleaved", 1, torch.float32, True, True),
    (33003, 1, 1, 128, 128, "half", 2, torch.bfloat16, False, True),
]


@pytest.mark.parametrize("case", MANY_TOKENS, ids=[str(i) for i in range(len(MANY_TOKENS))])
def test_qk_norm_rotary_of_many_tokens(K, Fn, case):
  test_qk_norm_rotary(K, Fn, case)
