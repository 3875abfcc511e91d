"""``ops.expert_gated_mlp``: the PyTorch form and the refusals on the CPU, the kernels against a
64-bit formulation on a GPU.

Tolerances of the bf16 kernels. Every rounding to bf16 is off by at most 2^-8 of the value it rounds.
The output: h is rounded (2^-8 sum |h w| at most), then y (2^-8 |y|). dx and the input weights'
gradient: the saved factor and dg / du are rounded (2 * 2^-8 of the sum of magnitudes), then the
result. The output weights' gradient: h, then the result. Accumulation in fp32 and the activation's
ex2 and rcp (2^-22) are covered by a tenth of one step more. "Sum of magnitudes" is the same product
evaluated with absolute values.
"""
import pytest
import torch
import torch.nn.functional as F

from vmoe_b200 import ops

gpu = pytest.mark.gpu
STEP = 2.0 ** -8


def make(e, r, h, m, o=None, bias=True, residual=False, dtype=torch.float32, wtype=None, seed=0,
         device="cpu"):
  g = torch.Generator().manual_seed(seed)
  o = o or h
  wtype = wtype or dtype
  rnd = lambda *s, scale=1.0, dt=wtype: (torch.randn(*s, generator=g) * scale).to(dt).to(device)
  return dict(x=rnd(e, r, h, dt=dtype), w_in=rnd(e, 2, m, h, scale=1.3 * h ** -0.5),
              b_in=rnd(e, 2, m, scale=0.3) if bias else None,
              w_out=rnd(e, o, m, scale=m ** -0.5), b_out=rnd(e, o, scale=0.3) if bias else None,
              residual=rnd(e, r, o, dt=dtype) if residual else None)


def split(t):
  return t["x"], t["w_in"], t["b_in"], t["w_out"], t["b_out"]


def oracle(t, act, dy=None, rounded_weights=True):
  """Output, gradients and the magnitudes that bound their rounding, in 64 bits."""
  d = {k: None if v is None else v.detach().cpu() for k, v in t.items()}
  if rounded_weights:  # the kernels' operands are the bf16 copies of fp32 master weights
    for k in ("w_in", "w_out"):
      d[k] = d[k].to(torch.bfloat16)
  d = {k: None if v is None else v.double() for k, v in d.items()}
  x, wg, wu, wo = d["x"], d["w_in"][:, 0], d["w_in"][:, 1], d["w_out"]
  g, u = x @ wg.transpose(1, 2), x @ wu.transpose(1, 2)
  if d["b_in"] is not None:
    g, u = g + d["b_in"][:, None, 0], u + d["b_in"][:, None, 1]
  g = g.requires_grad_()
  a = F.silu(g) if act == "silu" else F.gelu(g, approximate="tanh")
  (slope,) = torch.autograd.grad(a.sum(), g)
  a = a.detach()
  hid = a * u
  y = hid @ wo.transpose(1, 2)
  if d["b_out"] is not None:
    y = y + d["b_out"][:, None]
  if d["residual"] is not None:
    y = y + d["residual"]
  out = {"y": (y, hid.abs() @ wo.abs().transpose(1, 2))}
  if dy is not None:
    dy = dy.detach().cpu().double()
    dh = dy @ wo
    dg, du = dh * u * slope, dh * a
    tr = lambda v: v.transpose(1, 2)
    out["x"] = (dg @ wg + du @ wu, 2 * (dg.abs() @ wg.abs() + du.abs() @ wu.abs()))
    out["w_in"] = (torch.stack([tr(dg) @ x, tr(du) @ x], 1),
                   2 * torch.stack([tr(dg).abs() @ x.abs(), tr(du).abs() @ x.abs()], 1))
    out["w_out"] = (tr(dy) @ hid, tr(dy).abs() @ hid.abs())
    out["b_in"] = (torch.stack([dg.sum(1), du.sum(1)], 1),
                   2 * torch.stack([dg.abs().sum(1), du.abs().sum(1)], 1))
    out["b_out"] = (dy.sum(1), 0 * dy.sum(1))
    out["residual"] = (dy, 0 * dy)
  return out


def check(got, want, what, exact_type=False):
  value, magnitude = want
  far = (got.detach().cpu().double() - value).abs()
  bound = 1.1 * STEP * (magnitude + (0 if exact_type else value.abs())) + 1e-6
  assert got.shape == value.shape
  assert bool((far <= bound).all()), (what, float(far.max()), float((far / bound).max()))
  # The bound is a worst case of aligned errors; independent ones (each 0.42 steps in the mean square,
  # three of them at most) stay far below it once there are enough values.
  if value.numel() < 1000:
    return
  assert float(far.norm()) <= 1.2 * STEP * float(value.norm()) + 1e-6, what


def run(t, act, seed=5):
  names = [k for k in ("x", "w_in", "b_in", "w_out", "b_out", "residual") if t[k] is not None]
  leaves = {k: None if v is None else v.detach().requires_grad_() for k, v in t.items()}
  y = ops.expert_gated_mlp(*split(leaves), act=act, residual=leaves["residual"])
  g = torch.Generator().manual_seed(seed)
  dy = torch.randn(y.shape, generator=g).to(y.dtype).to(y.device)
  grads = torch.autograd.grad(y, [leaves[k] for k in names], dy)
  return y, dy, dict(zip(names, grads))


# ------------------------------------------------------------------------------------- CPU
@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("e,r,h,m,o,bias,residual", [
    (1, 5, 12, 20, None, True, False), (3, 4, 8, 16, 10, False, True), (2, 1, 7, 9, None, True, True),
    (2, 0, 8, 8, None, True, False)])
def test_pytorch_form(e, r, h, m, o, bias, residual, act):
  t = make(e, r, h, m, o, bias, residual, torch.float64)
  y, dy, grads = run(t, act)
  want = oracle(t, act, dy, rounded_weights=False)
  torch.testing.assert_close(y, want["y"][0])
  for k, g in grads.items():
    torch.testing.assert_close(g, want[k][0])


def test_gradient_against_differences():
  t = make(2, 3, 6, 5, dtype=torch.float64)
  leaves = [v.requires_grad_() for v in split(t)]
  for act in ("gelu", "silu"):
    assert torch.autograd.gradcheck(lambda *a: ops.expert_gated_mlp(*a, act=act), leaves)


@pytest.mark.parametrize("change,error", [
    (dict(act="relu"), ValueError), (dict(act=None), ValueError),
    (dict(x=torch.zeros(4, 8)), ValueError), (dict(x=torch.zeros(2, 4, 9)), ValueError),
    (dict(x=torch.zeros(3, 4, 8)), ValueError), (dict(w_in=torch.zeros(2, 3, 16, 8)), ValueError),
    (dict(w_in=torch.zeros(2, 16, 8)), ValueError), (dict(w_out=torch.zeros(2, 8, 15)), ValueError),
    (dict(b_in=torch.zeros(2, 16)), ValueError), (dict(b_out=torch.zeros(8)), ValueError),
    (dict(residual=torch.zeros(2, 4, 7)), ValueError),
    (dict(residual=torch.zeros(2, 4, 8, dtype=torch.float64)), TypeError),
    (dict(b_in=torch.zeros(2, 2, 16, dtype=torch.int32)), TypeError),
    (dict(w_in=torch.zeros(2, 2, 0, 8), w_out=torch.zeros(2, 8, 0), b_in=None), ValueError)])
def test_refusals(change, error):
  t = make(2, 4, 8, 16)
  t["act"] = "gelu"
  t.update(change)
  act = t.pop("act")
  with pytest.raises(error):
    ops.expert_gated_mlp(*split(t), act=act, residual=t["residual"])


# ------------------------------------------------------------------------------------- GPU
SHAPES = [
    # e, r, h, m, o, bias, residual
    (1, 1, 64, 64, None, True, True),
    (1, 1, 768, 2048, None, True, True),
    (3, 2, 128, 200, None, True, False),
    (1, 7, 136, 264, 72, False, True),
    (2, 16, 200, 328, None, True, True),
    (1, 17, 384, 136, None, True, False),
    (4, 33, 72, 1000, None, False, False),
    (1, 129, 256, 256, None, True, True),
    (2, 257, 264, 520, None, True, False),
    (1, 777, 320, 3416, None, True, True),
    (8, 300, 192, 776, None, True, False),
    (1, 2600, 128, 1024, 264, True, True),
    (8, 52, 128, 344, None, True, True),
    (3, 64, 192, 264, 136, True, False),
    (5, 100, 64, 72, None, False, True),
    (1, 1285, 256, 680, 1280, True, True),
    (1, 400, 520, 2048, None, True, False),
    (32, 3, 136, 344, None, True, True),
    (20, 11, 328, 264, 400, False, False),
]


@gpu
@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("e,r,h,m,o,bias,residual", SHAPES)
def test_kernels(e, r, h, m, o, bias, residual, act):
  t = make(e, r, h, m, o, bias, residual, torch.bfloat16, device="cuda")
  y, dy, grads = run(t, act)
  want = oracle(t, act, dy)
  assert y.dtype == torch.bfloat16
  check(y, want["y"], "y")
  for k, g in grads.items():
    assert g.dtype == t[k].dtype
    check(g, want[k], "d" + k)
  with torch.no_grad():  # the path without saved factors
    y2 = ops.expert_gated_mlp(*split(t), act=act, residual=t["residual"])
  assert torch.equal(y, y2)


@gpu
@pytest.mark.parametrize("e,r,h,m,o", [(1, 5, 33, 50, None), (2, 140, 100, 67, 30), (1, 1, 8, 1, 1)])
def test_odd_widths(e, r, h, m, o):
  t = make(e, r, h, m, o, True, True, torch.bfloat16, device="cuda")
  y, dy, grads = run(t, "gelu")
  want = oracle(t, "gelu", dy)
  check(y, want["y"], "y")
  for k, g in grads.items():
    check(g, want[k], "d" + k)


@gpu
def test_fp32_master_weights_and_bound_gradients():
  t = make(2, 150, 128, 264, dtype=torch.bfloat16, wtype=torch.float32, device="cuda")
  y, dy, grads = run(t, "silu")
  want = oracle(t, "silu", dy)
  check(y, want["y"], "y")
  for k in ("w_in", "w_out", "b_in", "b_out"):
    assert grads[k].dtype == torch.float32
    check(grads[k], want[k], "d" + k, exact_type=True)
  # Gradients that are bound to buffers already are added to, twice here.
  leaves = {k: t[k].detach().clone().requires_grad_() for k in ("w_in", "w_out", "b_in", "b_out")}
  for v in leaves.values():
    v.grad = torch.zeros_like(v)
  for _ in range(2):
    y = ops.expert_gated_mlp(t["x"], leaves["w_in"], leaves["b_in"], leaves["w_out"], leaves["b_out"],
                             act="silu")
    y.backward(dy)
  for k, v in leaves.items():
    torch.testing.assert_close(v.grad, 2 * grads[k], rtol=1e-5, atol=1e-5)


@gpu
def test_frozen_parts_and_layouts():
  t = make(2, 40, 64, 136, dtype=torch.bfloat16, residual=True, device="cuda")
  want, dy = None, torch.randn(2, 40, 64, device="cuda").bfloat16()
  want = oracle(t, "gelu", dy)
  for only in ("x", "w_in", "b_in", "w_out", "b_out", "residual"):
    leaves = dict(t)
    leaves[only] = t[only].detach().clone().requires_grad_()
    y = ops.expert_gated_mlp(*split(leaves), residual=leaves["residual"])
    (g,) = torch.autograd.grad(y, [leaves[only]], dy)
    check(g, want[only], only)
  # Transposed and strided operands, an expanded output gradient.
  x = t["x"].transpose(0, 1).contiguous().transpose(0, 1)
  res = torch.stack([t["residual"]] * 2, -1)[..., 0]
  w_in = t["w_in"].transpose(2, 3).contiguous().transpose(2, 3)
  y = ops.expert_gated_mlp(x, w_in, t["b_in"], t["w_out"], t["b_out"], residual=res)
  check(y, want["y"], "y")
  xg = x.detach().requires_grad_()
  ops.expert_gated_mlp(xg, w_in, t["b_in"], t["w_out"], t["b_out"], residual=res).sum().backward()
  check(xg.grad, oracle(t, "gelu", torch.ones(2, 40, 64))["x"], "dx")


@gpu
def test_no_rows():
  t = make(2, 0, 64, 72, dtype=torch.bfloat16, residual=True, device="cuda")
  y, _, grads = run(t, "gelu")
  assert y.shape == (2, 0, 64)
  for k in ("w_in", "w_out", "b_in", "b_out"):
    assert grads[k].shape == t[k].shape and not bool(grads[k].any())


@gpu
@pytest.mark.parametrize("r", [3, 300])
def test_results_do_not_depend_on_the_run(r):
  t = make(3, r, 256, 520, dtype=torch.bfloat16, device="cuda")
  first = run(t, "gelu")
  for _ in range(5):
    again = run(t, "gelu")
    assert torch.equal(first[0], again[0])
    for k in ("x", "w_in", "b_in", "w_out"):
      assert torch.equal(first[2][k], again[2][k]), k


@gpu
@pytest.mark.parametrize("r", [1, 200])
def test_side_stream_and_graph_replay(r):
  t = make(1, r, 128, 264, dtype=torch.bfloat16, residual=True, device="cuda")
  other = torch.randn_like(t["x"])
  want = {"a": run(t, "gelu"), "b": run(dict(t, x=other), "gelu")}
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    y = run(t, "gelu")[0]
  torch.cuda.current_stream().wait_stream(side)
  assert torch.equal(y, want["a"][0])
  buf = {k: v.clone() for k, v in t.items()}
  dy = want["a"][1]

  def step():
    leaves = {k: v.detach().requires_grad_() for k, v in buf.items()}
    y = ops.expert_gated_mlp(*split(leaves), residual=leaves["residual"])
    return (y,) + torch.autograd.grad(y, [leaves["x"], leaves["w_in"]], dy)

  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    step()
  torch.cuda.current_stream().wait_stream(side)
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    out = step()
  for key, src in (("b", other), ("a", t["x"])):
    buf["x"].copy_(src)
    graph.replay()
    assert torch.equal(out[0], want[key][0])
    assert torch.equal(out[1], want[key][2]["x"]) and torch.equal(out[2], want[key][2]["w_in"])


@gpu
@pytest.mark.parametrize("r", [2, 60])
def test_second_derivatives_are_refused(r):
  t = make(1, r, 64, 96, dtype=torch.bfloat16, device="cuda")
  x = t["x"].requires_grad_()
  y = ops.expert_gated_mlp(x, *split(t)[1:])
  (grad,) = torch.autograd.grad(y.sum(), x, create_graph=True)
  with pytest.raises(RuntimeError):
    grad.sum().backward()


@gpu
def test_offsets_past_32_bits():
  """The last rows where hidden units and factors have more than 2^31 elements."""
  t = make(1, 64, 64, 1024, dtype=torch.bfloat16, device="cuda")
  dy = torch.randn(1, 64, 64, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
  want = oracle(t, "gelu", dy)
  copies = 33000
  x = t["x"].repeat(1, copies, 1).requires_grad_()
  assert x.shape[1] * 1024 > 2 ** 31
  y = ops.expert_gated_mlp(x, *split(t)[1:])
  check(y[:, -64:], want["y"], "y")
  (dx,) = torch.autograd.grad(y, x, dy.repeat(1, copies, 1))
  check(dx[:, -64:], want["x"], "dx")
  check(dx[:, :64], want["x"], "dx")


@gpu
@pytest.mark.parametrize("e,r,h,m,o,bias,residual", [
    (1, 17, 64, 72, None, True, True), (1, 24, 384, 1000, 200, True, False),
    (1, 32, 520, 264, 72, False, True), (2, 31, 136, 328, None, True, True),
    (5, 25, 72, 64, 128, True, True), (1, 32, 8, 8, None, True, False)])
def test_rows_between_the_kernels(e, r, h, m, o, bias, residual):
  for act in ("gelu", "silu"):
    t = make(e, r, h, m, o, bias, residual, torch.bfloat16, device="cuda")
    y, dy, grads = run(t, act)
    want = oracle(t, act, dy)
    check(y, want["y"], "y")
    for k, g in grads.items():
      check(g, want[k], "d" + k)
