"""The multi-head attention block inside the networks that call it: forward and gradients against the chain in 64 bits,
a BigGAN training step with it, captured and eager."""
import math

import pytest
import torch

from tests import gan_util as U

pytestmark = pytest.mark.gpu

HB = 2.0 ** -8


@pytest.fixture(autouse=True)
def clean_config():
  from compare_gan_amd import gin
  gin.clear_config()
  yield
  gin.clear_config()


@pytest.mark.parametrize("n,h,w,c,heads,kv_heads,width", [(2, 8, 8, 64, None, None, 64), (3, 4, 6, 96, 4, 2, 32),
                                                        (1, 5, 5, 32, 2, 1, 16)])
def test_block_against_the_chain(dev, n, h, w, c, heads, kv_heads, width):
  """Relative error of whole tensors: the input of each of the five stages (projection, norm + rotation, attention,
  back projection, residual) and of their gradients is rounded to bf16, half a step of 2^-8 each, and the projections'
  operand images are bf16 too: seven roundings, uncorrelated over the sums."""
  from compare_gan_amd.architectures import arch_ops as ops
  gen = torch.Generator().manual_seed(n + c)
  store = ops.VariableStore(dev, seed=1)
  x = torch.randn((n, h, w, c), generator=gen).bfloat16().to(dev).requires_grad_(True)
  with ops.use_store(store):
    ops.attention_block(x.detach(), "att", False, kind="multi_head", num_heads=heads, num_kv_heads=kv_heads,
                        head_width=width)
    with torch.no_grad():
      for name, v in store.vars.items():      # weights of size 1 / sqrt(fan in), a sigma that shows
        if name.endswith("kernel"):
          v.copy_(torch.randn(v.shape, generator=gen).to(dev) / math.sqrt(v.shape[2]))
        elif name.endswith("gain"):
          v.copy_((1 + 0.2 * torch.randn(v.shape, generator=gen)).to(dev))
        else:
          v.fill_(0.7)
    out = ops.attention_block(x, "att", False, kind="multi_head", num_heads=heads, num_kv_heads=kv_heads,
                              head_width=width)
  dout = torch.randn((n, h, w, c), generator=gen).bfloat16().to(dev)
  names = sorted(store.vars)
  grads = torch.autograd.grad(out, [x] + [store.vars[k] for k in names], dout)
  heads = heads or max(1, c // width)
  kv_heads = kv_heads or heads
  v64 = {k.split("att/")[1]: store.vars[k].detach().double().cpu().requires_grad_(True) for k in names}
  x64 = x.detach().double().cpu().requires_grad_(True)
  rows = x64.reshape(n, h * w, c)
  half = width // 4
  f = 100.0 ** (-torch.arange(half, dtype=torch.float64) / half)
  cell = torch.arange(h * w)
  angle = torch.cat(((cell // w)[:, None] * f, (cell % w)[:, None] * f), 1)[None, :, None]

  def norm_turn(t, gain):
    t = t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-6) * gain
    a, b = t[..., :width // 2], t[..., width // 2:]
    return torch.cat((a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()), -1)
  q = norm_turn((rows @ v64["conv2d_q/kernel"][0, 0]).reshape(n, h * w, heads, width), v64["q_gain"])
  k = norm_turn((rows @ v64["conv2d_k/kernel"][0, 0]).reshape(n, h * w, kv_heads, width), v64["k_gain"])
  v = (rows @ v64["conv2d_v/kernel"][0, 0]).reshape(n, h * w, kv_heads, width)
  k, v = (t.repeat_interleave(heads // kv_heads, 2) for t in (k, v))
  p = torch.softmax(torch.einsum("nqhd,nkhd->nhqk", q, k) / math.sqrt(width), -1)
  o = torch.einsum("nhqk,nkhd->nqhd", p, v).reshape(n, h * w, heads * width)
  want = x64 + (v64["sigma"] * (o @ v64["conv2d_o/kernel"][0, 0])).reshape(n, h, w, c)
  wgrads = torch.autograd.grad(want, [x64] + [v64[k.split("att/")[1]] for k in names], dout.double().cpu())
  # sigma's gradient is one sum of n h w c terms of either sign, each off by its own relative roundings: its error is to
  # be held against the norm of the terms, not against what their signs leave of the sum
  terms = float((dout.double().cpu() * (o @ v64["conv2d_o/kernel"][0, 0]).reshape(n, h, w, c)).norm().detach())
  for name, a, b in zip(["out", "dx"] + names, (out,) + grads, (want,) + wgrads):
    a, b = a.detach().double().cpu(), b.detach()
    assert float((a - b).norm()) <= 7 * HB * (terms if name == "att/sigma" else float(b.norm())), name


@pytest.mark.parametrize("arch", ["resnet_biggan", "resnet_biggan_deep"])
def test_biggan_step_with_several_heads(dev, arch):
  """biggan_imagenet128.gin with the multi-head block: a captured step is the eager one to the bit, losses are finite
  and the block's variables get gradients (Adam moves them)."""
  bsz = 2
  bindings = ("options.batch_size = %d" % bsz, 'attention_block.kind = "multi_head"', "attention_block.num_heads = 4",
              "attention_block.num_kv_heads = 2", "attention_block.head_width = 32")
  if arch == "resnet_biggan":
    bindings += ("resnet_biggan.Generator.ch = 32", "resnet_biggan.Discriminator.ch = 32")
  else:
    bindings += ('options.architecture = "resnet_biggan_deep_arch"', "resnet_biggan_deep.Generator.ch = 32",
                 "resnet_biggan_deep.Discriminator.ch = 32", "G.batch_norm_fn = @conditional_batch_norm")
  eager, options, dataset = U.build_product("biggan_imagenet128.gin", bsz, dev, seed=5, bindings=bindings)
  graph, _, _ = U.build_product("biggan_imagenet128.gin", bsz, dev, seed=5, bindings=bindings)
  it = dataset.train_batches(bsz * (options["disc_iters"] + 1), seed=21)
  batches = [next(it) for _ in range(2)]
  with torch.no_grad():       # sigma = 0 in front of a fresh block: its projections would see no gradient
    for gan in (eager, graph):
      for name, v in gan.store.vars.items():
        if name.endswith("non_local_block/sigma"):
          v.fill_(0.5)
  before = {k: v.detach().clone() for k, v in eager.store.vars.items() if "non_local_block" in k}
  assert any(k.endswith("q_gain") for k in before)
  run = graph.capture_train_step()
  for images, labels in batches:
    x, y = torch.from_numpy(images).to(dev), torch.from_numpy(labels).to(dev)
    oe, og = eager.train_step(x, y), run(x, y)
    assert torch.isfinite(oe["g_loss"]).all() and torch.equal(oe["g_loss"], og["g_loss"])
  torch.cuda.synchronize()
  se, sg = eager.state_dict(), graph.state_dict()
  assert not [k for k in se if not torch.equal(se[k], sg[k])]
  still = [k for k, v in before.items() if k in eager.store.trainable and torch.equal(v, eager.store.vars[k])]
  assert not still, still


def test_block_captured_while_other_shapes_come_and_go(dev):
  """What a captured call reads stays where it is: replays agree with eager calls after many other shapes.  A shape that
  is first met inside a capture is refused with a message."""
  from compare_gan_amd.architectures import arch_ops as ops
  from compare_gan_amd.hip import functional as Fn
  side = 12
  rows = side * side
  gen = torch.Generator().manual_seed(5)
  q, k, v = (torch.randn((rows, 2, 32), generator=gen).bfloat16().to(dev) for _ in range(3))

  def call():
    positions, table, plan = ops._attention_constants(1, side, side, 2, 2, 32, 100.0, dev)
    a, b = Fn.qk_norm_rotary(q, k, None, None, positions, table)
    return Fn.packed_attention(a, b, v, plan)
  call()
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    held = call()
    with pytest.raises(RuntimeError, match="run it once before"):
      ops._attention_constants(1, side, side + 1, 2, 2, 32, 100.0, dev)
  others = []
  for n in range(2, 2 * ops.ATTENTION_SHAPES):
    ops._attention_constants(n, side, side, 2, 2, 32, 100.0, dev)
    others.append(torch.full((rows * 2,), -1, dtype=torch.int32, device=dev))
  for _ in range(3):
    q.copy_(torch.randn(q.shape, generator=gen))
    want = call()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, want)


@pytest.mark.parametrize("n,h,w,c,heads,kv_heads,width", [(2, 8, 8, 64, 1, 1, 64), (3, 4, 6, 96, 4, 2, 32),
                                                        (1, 5, 5, 32, 2, 1, 16)])
def test_block_with_independent_roundings(dev, n, h, w, c, heads, kv_heads, width):
  """The block against the chain in 64 bits with a bound that 2 % of a gradient does not pass.  Between an input and a
  gradient lie at most 16 roundings to bf16: the operand images of the four projections, q, k, v, the turned q and k, P,
  the attention's result, its incoming gradient, dS, the gradients of the turned and of the projected queries (keys), and
  the result's.  Each is an independent error of at most HB, HB / sqrt(3) root mean square, of what passes through:
  sqrt(16 / 3) HB = 0.9 % of the norm.  The gradients of sigma and of the gains are sums over rows of terms of either sign
  (of a key's gain: from rows of dS that sum to zero), each term off by its own roundings: their errors are held against
  the norm of the terms."""
  from compare_gan_amd.architectures import arch_ops as ops
  gen = torch.Generator().manual_seed(n + c)
  store = ops.VariableStore(dev, seed=1)
  x = torch.randn((n, h, w, c), generator=gen).bfloat16().to(dev).requires_grad_(True)
  args = dict(kind="multi_head", num_heads=heads, num_kv_heads=kv_heads, head_width=width)
  with ops.use_store(store):
    ops.attention_block(x.detach(), "att", False, **args)
    with torch.no_grad():
      for name, v in store.vars.items():
        if name.endswith("kernel"):
          v.copy_(torch.randn(v.shape, generator=gen).to(dev) / math.sqrt(v.shape[2]))
        elif name.endswith("gain"):
          v.copy_((1 + 0.2 * torch.randn(v.shape, generator=gen)).to(dev))
        else:
          v.fill_(0.7)
    out = ops.attention_block(x, "att", False, **args)
  dout = torch.randn((n, h, w, c), generator=gen).bfloat16().to(dev)
  names = sorted(store.vars)
  grads = torch.autograd.grad(out, [x] + [store.vars[k] for k in names], dout)
  rows, pairs = n * h * w, width // 2
  # gains and sigma with one entry for every term of their gradients
  shapes = {"q_gain": (rows, heads, width), "k_gain": (rows, kv_heads, width), "sigma": (rows, c)}
  v64 = {}
  for k in names:
    short, v = k.split("att/")[1], store.vars[k].detach().double().cpu()
    v64[short] = (v.expand(shapes[short]).clone() if short in shapes else v[0, 0].clone()).requires_grad_(True)
  x64 = x.detach().double().cpu().reshape(rows, c).requires_grad_(True)
  cell = torch.arange(rows) % (h * w)
  f = 100.0 ** (-torch.arange(pairs // 2, dtype=torch.float64) / (pairs // 2))
  z = torch.polar(torch.ones(rows, pairs, dtype=torch.float64),
                  torch.cat(((cell // w)[:, None] * f, (cell % w)[:, None] * f), 1))[:, None]

  def norm_turn(t, gain):
    t = t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-6) * gain
    t = torch.complex(t[..., :pairs], t[..., pairs:]) * z
    return torch.cat((t.real, t.imag), -1)

  def project(which, m):
    return (x64 @ v64["conv2d_%s/kernel" % which]).reshape(rows, m, width)
  q, k = norm_turn(project("q", heads), v64["q_gain"]), norm_turn(project("k", kv_heads), v64["k_gain"])
  v = project("v", kv_heads)
  o = torch.empty(0, heads * width, dtype=torch.float64)
  for i in range(n):
    mine = slice(i * h * w, (i + 1) * h * w)
    per_head = [torch.softmax(q[mine, j] @ k[mine, j * kv_heads // heads].t() / math.sqrt(width), -1) @
                v[mine, j * kv_heads // heads] for j in range(heads)]
    o = torch.cat((o, torch.cat(per_head, 1)))
  want = x64 + v64["sigma"] * (o @ v64["conv2d_o/kernel"])
  short = [k.split("att/")[1] for k in names]
  wgrads = torch.autograd.grad(want, [x64] + [v64[k] for k in short], dout.double().cpu().reshape(rows, c))
  for name, a, b in zip(["out", "dx"] + short, (out,) + grads, (want,) + wgrads):
    a, b = a.detach().double().cpu(), b.detach()
    size = float(b.norm())
    if name in shapes:
      b = b.reshape(-1, a.numel()).sum(0)
    assert float((a.flatten() - b.flatten()).norm()) <= math.sqrt(16 / 3) * HB * size, name
