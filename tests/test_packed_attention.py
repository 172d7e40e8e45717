"""Rotary tables, plans and refusals of the packed attention operators (no GPU)."""
import ctypes
import math

import numpy as np
import pytest
import torch

from compare_gan_amd.hip import _lib
from compare_gan_amd.hip import functional as Fn
from compare_gan_amd.hip import kernels as K


# -- frequencies ---------------------------------------------------------------------------------
@pytest.mark.parametrize("rot,axes", [(2, 1), (4, 2), (64, 1), (64, 2), (36, 3)])
@pytest.mark.parametrize("scaling,factor", [("none", 1.0), ("linear", 8.0), ("ntk", 4.0), ("yarn", 16.0)])
def test_rotary_table(rot, axes, scaling, factor):
  t = K.RotaryTable(rot, base=10000.0, scaling=scaling, factor=factor, original_length=2048, axes=axes,
                    device="cpu")
  assert t.freq.dtype == torch.float64 and t.freq.shape == (rot // 2,)
  n = rot // 2 // axes
  f = t.freq.numpy() * 2 * math.pi
  for a in range(1, axes):
    np.testing.assert_array_equal(f[:n], f[a * n:(a + 1) * n])
  plain = 10000.0 ** (-np.arange(n) / n)
  if scaling == "none":
    np.testing.assert_allclose(f[:n], plain, rtol=1e-14)
  elif scaling == "linear":
    np.testing.assert_allclose(f[:n], plain / factor, rtol=1e-14)
  elif scaling == "ntk":      # the fastest pair stays, the slowest is divided by the factor
    assert f[0] == pytest.approx(1.0, rel=1e-14)
    if n > 1:
      assert f[n - 1] == pytest.approx(plain[-1] / factor, rel=1e-12)
  else:
    turns = 2048 * plain / (2 * math.pi)
    for i in range(n):
      if turns[i] >= 32:
        assert f[i] == pytest.approx(plain[i], rel=1e-14)
      elif turns[i] <= 1:
        assert f[i] == pytest.approx(plain[i] / factor, rel=1e-14)
      else:
        assert plain[i] / factor < f[i] < plain[i]
  assert t.amplitude == (0.1 * math.log(factor) + 1.0 if scaling == "yarn" else 1.0)


@pytest.mark.parametrize("kw", [dict(rotary_dim=3), dict(rotary_dim=0), dict(rotary_dim=6, axes=2),
                                dict(rotary_dim=8, layout="pairs"), dict(rotary_dim=8, scaling="log"),
                                dict(rotary_dim=8, base=0.0), dict(rotary_dim=8, base=float("nan")),
                                dict(rotary_dim=8, scaling="linear", factor=0.5),
                                dict(rotary_dim=8, factor=float("inf")), dict(rotary_dim=8, axes=0),
                                dict(rotary_dim=8, original_length=0)])
def test_rotary_table_refusals(kw):
  with pytest.raises(ValueError):
    K.RotaryTable(device="cpu", **kw)


# -- plans ---------------------------------------------------------------------------------------
def _lists(plan):
  i = plan.info
  at = 4 * i.sequences
  out = {"seqs": plan.host[:at].reshape(-1, 4)}
  for name in ("tiles", "thin4", "thin1", "joins", "dq_tiles", "dq_joins", "dkv_tiles", "dkv_joins", "small"):
    n = getattr(i, name)
    out[name] = plan.host[at:at + 8 * n].reshape(n, 8)
    at += 8 * n
  assert at == i.ints
  return out


PLANS = [
    ("one token", [1], None, 1, 1, False, None),
    ("ragged", [2047, 1, 0, 5000, 333, 64, 129], None, 8, 2, True, None),
    ("maps", [256] * 40, None, 3, 3, False, None),
    ("new tokens", [1] * 5, [1, 8192, 0, 777, 40000], 32, 8, True, 40000),
    ("few rows, many keys", [200], [70001], 2, 1, False, None),
    ("queries in front of the keys", [100, 40], [30, 0], 4, 4, True, None),
    ("odd heads", [33, 65, 31], [64, 1, 300], 15, 3, True, 512),
    ("few small beside large", [3] * 128 + [200], None, 2, 2, True, None),
    ("many small beside large", [3] * 129 + [200, 0], None, 2, 2, True, None),
    ("many new tokens, few long", [1] * 300, [5] * 299 + [900], 4, 1, True, 1000),
    ("one row a head, 40 shared", [1], [3000], 40, 1, False, None),
]


@pytest.mark.parametrize("case", PLANS, ids=[c[0] for c in PLANS])
def test_plan_covers_every_row_and_key_once(case):
  _, q, k, heads, kv_heads, causal, capacity = case
  kk = q if k is None else k
  starts = None if capacity is None else [i * capacity for i in range(len(kk))]
  plan = K.AttentionPlan(q, k, heads=heads, kv_heads=kv_heads, causal=causal, k_starts=starts, device="cpu")
  p, g = _lists(plan), heads // kv_heads
  assert p["seqs"][:, 1].tolist() == list(q) and p["seqs"][:, 3].tolist() == list(kk)
  assert plan.q_rows == sum(q) and plan.q_dense
  assert plan.k_rows == max([s + n for s, n in zip(p["seqs"][:, 2].tolist(), kk) if n] + [0])

  def seen(b, token):            # keys of a token
    return max(0, min(kk[b], token + kk[b] - q[b] + 1)) if causal else kk[b]

  used = set()
  pieces = {}
  for name, tile, step in (("tiles", 128, 64), ("thin4", 32, 32), ("thin1", 32, 32)):
    for b, h, row0, k0, k1, part, _, _ in p[name].tolist():
      rows = q[b] * g
      assert 0 <= h < kv_heads and row0 % tile == 0 and row0 < rows
      # few rows and keys: in a form of their own only where they are many or alone
      assert (rows > 32) == (name == "tiles") or (name == "tiles" and k1 <= 128 and part < 0)
      assert 0 <= k0 <= k1 <= kk[b] and k0 % step == 0
      pieces.setdefault((b, h, row0), []).append((k0, k1, part))
      if part >= 0:
        units = tile // 32
        assert not used & set(range(part, part + units))
        used |= set(range(part, part + units))
  assert len(p["thin1"]) == 0 or len(p["thin1"]) > 256 or not len(p["thin4"]) + len(p["tiles"])
  assert len(used) == plan.info.parts and (not used or max(used) == plan.info.parts - 1)
  joins = {(b, h, r): (n, parts, unit, units) for b, h, r, n, parts, unit, units, _ in p["joins"].tolist()}
  for b, n in enumerate(q):
    for h in range(kv_heads):
      tile = 128 if n * g > 32 else 32
      for r in range(0, n * g, tile):
        got = sorted(pieces.pop((b, h, r)))
        end = seen(b, (min(r + tile, n * g) - 1) // g)
        assert got[0][0] == 0 and got[-1][1] == end
        assert all(x[1] == y[0] for x, y in zip(got, got[1:]))
        if len(got) == 1:
          assert got[0][2] == -1 and (b, h, r) not in joins
        else:
          rows, parts, unit, units = joins.pop((b, h, r))
          assert rows == min(tile, n * g - r) and units == tile // 32
          assert [x[2] for x in got] == [unit + i * units for i in range(parts)]
  assert not pieces and not joins
  # gradients: sequences that fit one wave as a whole, the others in tiles whose parts follow one another
  alone = sorted((b, h) for b, h, _, _, k1, _, _, _ in p["small"].tolist())
  one_wave = [q[b] * g <= 32 and kk[b] <= 32 for b in range(len(q))]
  own_form = all(one_wave) or kv_heads * sum(f and q[b] + kk[b] > 0 for b, f in enumerate(one_wave)) > 256
  fits = lambda b: own_form and one_wave[b]
  assert alone == sorted((b, h) for b in range(len(q)) for h in range(kv_heads) if fits(b) and (q[b] or kk[b]))
  want_q, want_k = {}, {}
  for b in range(len(q)):
    for h in range(kv_heads):
      if fits(b):
        continue
      for r in range(0, q[b] * g, 128):
        want_q[(b, h, r)] = (0, seen(b, (min(r + 128, q[b] * g) - 1) // g), min(128, q[b] * g - r))
      for key in range(0, kk[b], 128):
        first = 0
        while first < q[b] and seen(b, first) <= key:
          first += 1
        want_k[(b, h, key)] = (first * g, q[b] * g, min(128, kk[b] - key))
  for tiles, joins, want, total in (("dq_tiles", "dq_joins", want_q, plan.info.dq_parts),
                                    ("dkv_tiles", "dkv_joins", want_k, plan.info.dkv_parts)):
    pieces, joined = {}, {}
    for b, h, at, x0, x1, part, _, _ in p[tiles].tolist():
      pieces.setdefault((b, h, at), []).append((x0, x1, part))
    for b, h, at, n, parts, first, _, _ in p[joins].tolist():
      joined[(b, h, at)] = (n, parts, first)
    assert sorted(pieces) == sorted(want)
    numbers = []
    for key, got in pieces.items():
      got.sort()
      start, end, n = want[key]
      assert got[0][0] == start and got[-1][1] == end and all(x[1] == y[0] for x, y in zip(got, got[1:]))
      if len(got) == 1:
        assert got[0][2] == -1 and key not in joined
      else:
        first = joined[key][2]
        assert joined.pop(key) == (n, len(got), first)
        assert [x[2] for x in got] == list(range(first, first + len(got)))
        numbers += [x[2] for x in got]
    assert not joined and sorted(numbers) == list(range(total))


def test_plan_spreads_few_rows_over_the_chip():
  plan = K.AttentionPlan([1] * 4, [50000] * 4, heads=8, kv_heads=2, causal=True, device="cpu")
  p = _lists(plan)
  assert len(p["thin4"]) >= 512 and len(p["joins"]) == 8
  assert max(k1 - k0 for _, _, _, k0, k1, _, _, _ in p["thin4"].tolist()) <= 1024


@pytest.mark.parametrize("kw", [
    dict(q_lengths=[]), dict(q_lengths=[-1]), dict(q_lengths=[4], k_lengths=[4, 4]),
    dict(q_lengths=[4], heads=3, kv_heads=2), dict(q_lengths=[4], heads=0),
    dict(q_lengths=[4, 4], q_starts=[0, 2]), dict(q_lengths=[4, 4], q_starts=[0]),
    dict(q_lengths=[4, 4], k_starts=[3, 0]), dict(q_lengths=[4], k_starts=[-1]),
    dict(q_lengths=[2.5]), dict(q_lengths=[4], k_starts=[0.5]), dict(q_lengths=[2 ** 30]), dict(q_lengths=[2 ** 40]), dict(q_lengths=[4], heads=8192)])
def test_plan_refusals(kw):
  with pytest.raises((ValueError, _lib.CgamdError)):
    K.AttentionPlan(device="cpu", **kw)


def test_plan_entry_point_refuses_without_throwing():
  lib = _lib.load()
  info = _lib.AttentionPlanInfo()
  one = np.ones(1, np.int32)
  p = one.ctypes.data
  assert lib.cg_host_attention_plan(None, p, p, p, 1, 1, 1, 0, None, 0, ctypes.byref(info)) == -1
  assert lib.cg_host_attention_plan(p, p, p, p, 0, 1, 1, 0, None, 0, ctypes.byref(info)) == -1
  assert lib.cg_host_attention_plan(p, p, p, p, 1, 3, 2, 0, None, 0, ctypes.byref(info)) == -1
  assert lib.cg_host_attention_plan(p, p, p, p, 1, 1, 1, 0, p, 1, ctypes.byref(info)) == -4
  neg = -one
  assert lib.cg_host_attention_plan(p, neg.ctypes.data, p, p, 1, 1, 1, 0, None, 0, ctypes.byref(info)) == -1


def test_entry_points_refuse_without_a_launch():
  """Pointers that are never followed: every refusal comes before the first launch."""
  lib = _lib.load()
  fake = 4096
  plan = K.AttentionPlan([4], heads=2, kv_heads=1, device="cpu")
  info = ctypes.byref(plan.info)

  def call(entry, **kw):
    f = dict(q=fake, k=fake, v=fake, q_stride_t=128, q_stride_h=64, k_stride_t=64, k_stride_h=64,
             v_stride_t=64, v_stride_h=64, q_rows=4, k_rows=4, D=64, Dv=64, scale=1.0)
    f.update(kw)
    arg = ctypes.byref(_lib.AttentionInput(*[f[n] for n, _ in _lib.AttentionInput._fields_]))
    if entry == "fwd":
      return lib.cg_packed_attention_fwd(arg, info, fake, None, None, None, None, 0, None)
    return lib.cg_packed_attention_bwd(arg, info, fake, fake, fake, fake, fake, fake, fake, fake, None, 0, None)
  for entry in ("fwd", "bwd"):
    assert call(entry, D=60) == -2 and call(entry, Dv=136) == -2 and call(entry, D=0) == -2
    assert call(entry, scale=0.0) == -1 and call(entry, scale=float("nan")) == -1
    assert call(entry, scale=float("inf")) == -1
    assert call(entry, q_rows=3) == -1 and call(entry, k_rows=3) == -1
    assert call(entry, k_stride_t=63) == -2 and call(entry, q_stride_t=-8) == -2
    assert call(entry, v=fake + 8) == -2 and call(entry, q=None) == -1
    assert call(entry, k_stride_t=2 ** 26) == -2
  assert call("fwd") == -1          # no output
  plan = K.AttentionPlan([100], heads=2, kv_heads=1, device="cpu")     # (4 rows need none)
  info = ctypes.byref(plan.info)
  assert call("bwd", q_rows=100, k_rows=100) == -4                     # no workspace
  rows = _lib.HeadRows(fake, 64, 64, 1, None)
  r = ctypes.byref(rows)
  rot = _lib.Rotation(fake, fake, 1.0, 1, 64, 0)
  wide = _lib.Rotation(fake, fake, 1.0, 2, 66, 0)
  assert lib.cg_rotary(r, 1, 63, 0, ctypes.byref(rot), 0, fake, None) == -2
  assert lib.cg_rotary(r, 1, 258, 0, ctypes.byref(rot), 0, fake, None) == -2
  assert lib.cg_rotary(r, 1, 64, 2, ctypes.byref(rot), 0, fake, None) == -2
  assert lib.cg_rotary(r, 1, 64, 0, ctypes.byref(wide), 0, fake, None) == -1
  assert lib.cg_rotary(r, 1, 64, 0, None, 0, fake, None) == -1
  assert lib.cg_rotary(r, 1, 64, 0, ctypes.byref(rot), 0, None, None) == -1
  assert lib.cg_qk_norm_rotary_fwd(r, None, 1, 64, 0, 1e-6, None, fake, fake, None) == -1
  assert lib.cg_qk_norm_rotary_fwd(r, r, 1, 64, 0, -1.0, None, fake, fake, None) == -1
  assert lib.cg_qk_norm_rotary_bwd(r, r, fake, fake, 1, 64, 0, 1e-6, None, fake, fake, fake, fake, None, 0,
                                   None) == -4


def test_operators_refuse_host_tensors():
  x = torch.zeros(2, 1, 8)
  pos = torch.zeros(2, dtype=torch.int32)
  table = K.RotaryTable(8, device="cpu")
  with pytest.raises(ValueError, match="GPU"):
    Fn.rotary(x, pos, table)
  with pytest.raises(ValueError, match="GPU"):
    Fn.qk_norm_rotary(x, x, None, None, pos, table)
  with pytest.raises(ValueError, match="GPU"):
    Fn.packed_attention(x.bfloat16(), x.bfloat16(), x.bfloat16(), K.AttentionPlan([2], device="cpu"))


def test_packed_structures_have_the_declared_layout():
  rows = torch.zeros(200).as_strided((3, 2, 8), (40, 16, 1))
  raw = _lib.HeadRows.from_buffer_copy(K._head_rows(rows, rows))
  assert (raw.x, raw.stride_t, raw.stride_h, raw.heads, raw.gain) == (rows.data_ptr(), 40, 16, 2, rows.data_ptr())
  table = K.RotaryTable(8, scaling="yarn", factor=2.0, axes=2, layout="interleaved", device="cpu")
  raw = _lib.Rotation.from_buffer_copy(table.packed(rows))
  assert (raw.positions, raw.freq, raw.axes, raw.rot, raw.interleaved) == (
      rows.data_ptr(), table.freq.data_ptr(), 2, 8, 1)
  assert raw.amplitude == pytest.approx(table.amplitude, rel=1e-7)
  raw = _lib.AttentionInput.from_buffer_copy(K._attention_packed(rows, rows[:2], rows[:1], 0.5))
  assert [getattr(raw, n) for n, _ in raw._fields_] == [rows.data_ptr()] * 3 + [40, 16, 40, 16, 0, 16, 3, 2, 8, 8, 0.5]


class _OnTheGpu(torch.Tensor):
  """A tensor without memory that the checks take for one on the GPU."""
  is_cuda = property(lambda self: True)

  def get_device(self):
    return 0


def _shape_only(shape, dtype=torch.bfloat16):
  return torch.empty(shape, dtype=dtype, device="meta").as_subclass(_OnTheGpu)


def test_rows_and_heads_beyond_32_bits_are_refused(monkeypatch):
  """Before anything is allocated or called: 2^32 rows would arrive as none, 2^32 + 5 as 5."""
  def called(*_):
    raise AssertionError("reached the library")
  monkeypatch.setattr(K, "_launch", called)
  table = K.RotaryTable(2, device="cpu")
  table.index = 0
  for rows, heads in ((2 ** 31, 1), (2 ** 32, 1), (2 ** 32 + 5, 1), (1, 2 ** 30), (1, 2 ** 32 + 1)):
    x, pos = _shape_only((rows, heads, 2)), _shape_only((rows,), torch.int32)
    few = _shape_only((rows, 1, 2))
    with pytest.raises(ValueError, match="rows and"):
      K.rotary(x, pos, table)
    with pytest.raises(ValueError, match="rows and"):
      Fn.qk_norm_rotary(few, x, None, None)
    with pytest.raises(ValueError, match="rows and"):
      K.qk_norm_rotary_bwd(x, few, None, None, None, None, x, few)
    with pytest.raises(ValueError, match="rows and"):
      Fn.packed_attention(x, few, few, K.AttentionPlan([1], device="cpu"))
  lib = _lib.load()
  rows = ctypes.byref(_lib.HeadRows(4096, 64, 64, 2 ** 30, None))
  rot = ctypes.byref(_lib.Rotation(4096, 4096, 1.0, 1, 64, 0))
  assert lib.cg_rotary(rows, 1, 64, 0, rot, 0, 4096, None) == -2
  assert lib.cg_qk_norm_rotary_fwd(rows, rows, 1, 64, 0, 1e-6, None, 4096, 4096, None) == -2


class _Recorder(object):
  """Stands for a constant's tensor: notes the streams that are recorded with the allocator."""

  def __init__(self):
    self.recorded = []

  def record_stream(self, stream):
    self.recorded.append(stream)


def test_constants_are_recorded_on_every_other_stream_that_reads_them(monkeypatch):
  """Once a stream, before the call, the one they were made on excepted; calls on other streams' handles stay apart."""
  current = {"raw": 7}
  calls = []

  class Library(object):
    def __getattr__(self, name):
      if name.endswith("workspace_bytes"):
        return lambda *_: 0
      return lambda *args: calls.append((name, args[-1], len(seen.recorded))) or 0
  x, pos = torch.zeros((4, 1, 8), dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int32)
  seen = _Recorder()
  table = K.RotaryTable(8, device="cpu")
  plan = K.AttentionPlan([40], device="cpu")
  monkeypatch.setattr(K, "lib", Library)
  monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: current["raw"], raising=False)
  monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
  monkeypatch.setattr(torch.cuda, "current_stream", lambda index=None: ("stream", current["raw"]))
  monkeypatch.setattr(torch.Tensor, "get_device", lambda self: 0)
  y = torch.zeros((40, 1, 8), dtype=torch.bfloat16)
  stats = torch.zeros((40, 1))
  entries = [(table, lambda: K._rotate(x, pos, table, False)),
             (table, lambda: K._qk_rows(x, x, None, None, pos, table, 1e-6)),
             (table, lambda: K._qk_grads(x, x, None, None, pos, table, x, x, 1e-6)),
             (plan, lambda: K._attention_rows(y, y, y, plan, 1.0, True)),
             (plan, lambda: K._attention_grads(y, y, y, plan, y, stats, y, y, 1.0))]
  for owner, call in entries:
    seen = _Recorder()
    owner.constant.tensor, owner.constant.streams = seen, {7}
    del calls[:]
    for raw in (7, 9, 9, 7, 11, 9):
      current["raw"] = raw
      call()
    assert seen.recorded == [("stream", 9), ("stream", 11)]
    assert [c[1:] for c in calls] == [(7, 0), (9, 1), (9, 1), (7, 1), (11, 2), (9, 2)]
  # nothing to keep: no table
  K._qk_rows(x, x, None, None, None, None, 1e-6)


@pytest.mark.parametrize("q_lengths,q_starts", [([2 ** 62 + 5], [2 ** 63 - 2 ** 32 + 10]), ([5], [2 ** 63 - 2]),
                                                ([2 ** 63 - 1, 3], None), ([2 ** 62, 2 ** 62, 4], None)])
def test_plan_refuses_lengths_whose_sums_wrap(q_lengths, q_starts):
  """Their low 32 bits are lengths and starts that a plan would take."""
  with pytest.raises(ValueError, match="2\\^30"):
    K.AttentionPlan(np.array(q_lengths), [3] * len(q_lengths), q_starts=None if q_starts is None else np.array(q_starts),
                    device="cpu")


@pytest.mark.parametrize("kw", [dict(scaling="yarn", factor=2.0, original_length=float("nan")),
                                dict(scaling="yarn", factor=2.0, original_length=float("inf")),
                                dict(scaling="ntk", base=1e300, factor=1e10), dict(scaling="ntk", factor=1e300),
                                dict(scaling="ntk", base=1e300, factor=1e300), dict(base=1e-320),
                                dict(scaling="ntk", base=1e-320)])
def test_rotary_table_refuses_what_has_no_frequencies(kw):
  with pytest.raises(ValueError):
    K.RotaryTable(8, device="cpu", **kw)


@pytest.mark.parametrize("kw", [dict(scaling="ntk", base=1e150, factor=1e100), dict(base=1e-299), dict(base=1e300)])
def test_rotary_table_at_the_ends_of_its_range(kw):
  f = K.RotaryTable(8, device="cpu", **kw).freq
  assert torch.isfinite(f).all() and (f > 0).all()


def test_attention_entry_points_refuse_what_is_not_aligned():
  """The plan is read and partial results are written 16 bytes at a time; strides whose products would wrap."""
  lib, fake = _lib.load(), 4096
  plan = K.AttentionPlan([200], [70001], heads=2, kv_heads=1, device="cpu")
  info = ctypes.byref(plan.info)
  need = lib.cg_packed_attention_fwd_workspace_bytes(info, 64)
  assert plan.info.parts > 0 and need > 0

  def call(data=fake, ws=fake, **kw):
    f = dict(q=fake, k=fake, v=fake, q_stride_t=128, q_stride_h=64, k_stride_t=64, k_stride_h=64,
             v_stride_t=64, v_stride_h=64, q_rows=200, k_rows=70001, D=64, Dv=64, scale=1.0)
    f.update(kw)
    arg = ctypes.byref(_lib.AttentionInput(*[f[n] for n, _ in _lib.AttentionInput._fields_]))
    return [lib.cg_packed_attention_fwd(arg, info, data, fake, None, None, ws, need if ws else 0, None),
            lib.cg_packed_attention_bwd(arg, info, data, fake, fake, fake, fake, fake, fake, fake, ws,
                                        0, None)]
  assert call(ws=None) == [-4, -4]
  assert call(data=fake + 4) == [-2, -2] and call(data=fake + 8) == [-2, -2]
  assert call(ws=fake + 8)[0] == -2
  for name in ("q_stride_t", "q_stride_h", "k_stride_t", "k_stride_h", "v_stride_t", "v_stride_h"):
    assert call(ws=None, **{name: 2 ** 61}) == [-2, -2], name


def test_shared_memory_is_seen():
  x = torch.zeros(10, 6, 16)
  whole = [(x[:, :2], x[:, 2:4], True), (x[:5], x[5:], False), (x[5:], x[:5], False), (x[:6], x[5:], True),
           (x[:1, :2], x[:1, 2:], False), (x, x.clone(), False), (x[3:4], x, True), (x[:0], x, False),
           (x[2, :1].expand(4, 16), x[2], True), (x[2, :1].expand(4, 16), x[2, 1:], False)]
  for a, b, want in whole:
    assert K._share_memory(a, b) is want and K._share_memory(b, a) is want
