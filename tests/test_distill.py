"""``losses.top_logits`` and ``losses.distill_xent``: the PyTorch forms and the refusals on the CPU,
the kernels against 64-bit formulas on a GPU.

Tolerances. fp32 results of the kernels: the exponent of a term is x c + a with x c, a and c each
rounded once (relative 2^-24, |x c| <= 64 here), so a probability is off by at most
3 * 64 * 2^-24 * ln 2 < 8e-6 and a log-sum-exp, relative to its size >= 1, by less than 1e-5; ex2's
2^-22 is far below. 16-bit gradients add half a step of their type (bf16 2^-8, fp16 2^-11).
"""
import math

import pytest
import torch

from vmoe_b200.ops import losses

gpu = pytest.mark.gpu
F32 = 1e-5
HALF_STEP = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(rows, n, dtype, seed=0, pad=0, device="cpu", scale=2.0):
  g = torch.Generator().manual_seed(seed)
  x = (torch.randn(rows, n + pad, generator=g) * scale).to(dtype)
  return x.to(device)[:, :n]


def top_oracle(x, k, temperature):
  """Order by (value, lower class first) through a sort of exact pairs; NaN above everything."""
  xd = x.detach().cpu().double()
  key = torch.where(torch.isnan(xd), torch.full_like(xd, math.inf), xd)
  nan = torch.isnan(xd)
  out_i, out_r = [], []
  for row, isnan in zip(key, nan):
    order = sorted(range(len(row)), key=lambda j: (not bool(isnan[j]), -float(row[j]), j))
    out_i.append(order[:k])
    others = torch.tensor(order[k:], dtype=torch.long)
    vals = torch.where(isnan[others], torch.full_like(row[others], math.nan), row[others])
    out_r.append(torch.logsumexp(vals / temperature, 0) if len(others) else
                 torch.tensor(-math.inf, dtype=torch.float64))
  return torch.tensor(out_i, dtype=torch.int32), torch.stack(out_r)


def distill_oracle(logits, values, indices, rest, temperature, dloss):
  """Loss and gradient from the definition, row by row, in 64 bits."""
  rows, n = logits.shape
  losses_, grads = [], []
  for r in range(rows):
    z = logits[r].detach().cpu().double() / temperature
    seen, t = [], []
    for v, i in zip(values[r].cpu().double().tolist(), indices[r].cpu().tolist()):
      if 0 <= i < n and i not in seen:
        seen.append(i)
        t.append(v / temperature)
    mask = torch.ones(n, dtype=torch.bool)
    mask[seen] = False
    outcomes = list(t) + ([float(rest[r])] if rest is not None else [])
    if not outcomes or max(outcomes) == -math.inf:
      losses_.append(0.0)
      grads.append(torch.zeros(n, dtype=torch.float64))
      continue
    log_p = torch.log_softmax(torch.tensor(outcomes, dtype=torch.float64), 0)
    p = log_p.exp()
    log_z = torch.log_softmax(z, 0)
    q = log_z.exp()
    log_q = log_z[seen]
    if rest is not None:
      log_q = torch.cat([log_q, torch.logsumexp(log_z[mask], 0).reshape(1)])
    terms = torch.where(p > 0, p * (log_p - log_q), torch.zeros_like(p))
    losses_.append(float(terms.sum()) * temperature ** 2)
    g = q.clone()
    if rest is not None:
      q_rest = q[mask].sum()
      if q_rest > 0:
        g[mask] *= 1 - p[-1] / q_rest
    for j, i in enumerate(seen):
      g[i] = q[i] - p[j]
    grads.append(g * temperature * float(dloss[r]))
  return torch.tensor(losses_, dtype=torch.float64), torch.stack(grads)


def teacher_of(x, k, temperature, seed=1, noise=1.0):
  t = (x.float() + noise * make(*x.shape, torch.float32, seed).to(x.device)).to(x.dtype)
  return losses.top_logits(t.cpu(), k, temperature=temperature)


# ------------------------------------------------------------------------------------- CPU
@pytest.mark.parametrize("rows,n,k,temperature", [(3, 17, 5, 1.0), (2, 8, 8, 2.0), (4, 1, 1, 1.0),
                                                  (1, 40, 1, 0.5)])
def test_top_logits_pytorch_form(rows, n, k, temperature):
  x = (make(rows, n, torch.float32) * 2).round() / 2  # many ties
  got = losses.top_logits(x, k, temperature=temperature)
  idx, rest = top_oracle(x, k, temperature)
  assert torch.equal(got.indices, idx) and got.indices.dtype == torch.int32
  assert torch.equal(got.values, x.gather(1, idx.long()))
  torch.testing.assert_close(got.rest.double(), rest, rtol=F32, atol=F32)


@pytest.mark.parametrize("with_rest", [False, True])
@pytest.mark.parametrize("temperature", [1.0, 3.0])
def test_distill_pytorch_form_and_its_gradient(with_rest, temperature):
  x = make(5, 23, torch.float64, scale=1.5).requires_grad_()
  t = teacher_of(x.detach().float(), 6, temperature)
  idx = t.indices.clone()
  idx[1, 4:] = -1
  idx[2, 3] = idx[2, 0]
  idx[3] = -1
  rest = t.rest if with_rest else None
  dloss = torch.tensor([1.0, -0.5, 2.0, 1.0, 0.0], dtype=torch.float64)
  loss = losses.distill_xent(x, t.values, idx, rest, temperature=temperature)
  (grad,) = torch.autograd.grad(loss, x, dloss.float())
  want, want_grad = distill_oracle(x, t.values, idx, rest, temperature, dloss)
  torch.testing.assert_close(loss.double(), want, rtol=F32, atol=F32)
  torch.testing.assert_close(grad, want_grad, rtol=F32, atol=F32)
  # The formula's gradient against central differences of the loss in 64 bits.
  eps = 1e-5
  step = torch.zeros_like(x)
  step[:, 7] = eps
  up, _ = distill_oracle(x.detach() + step, t.values, idx, rest, temperature, dloss)
  down, _ = distill_oracle(x.detach() - step, t.values, idx, rest, temperature, dloss)
  torch.testing.assert_close((up - down) / (2 * eps) * dloss, want_grad[:, 7], rtol=1e-6, atol=1e-8)


def test_a_student_that_equals_its_teacher_has_no_loss():
  x = make(4, 50, torch.float32)
  t = losses.top_logits(x, 7, temperature=2.0)
  loss = losses.distill_xent(x, *t, temperature=2.0)
  assert float(loss.abs().max()) < 1e-6


@pytest.mark.parametrize("call,error", [
    (lambda x, v, i: losses.top_logits(x[0], 2), ValueError),
    (lambda x, v, i: losses.top_logits(x, 0), ValueError),
    (lambda x, v, i: losses.top_logits(x, 21), ValueError),
    (lambda x, v, i: losses.top_logits(x.repeat(1, 20), 257), ValueError),
    (lambda x, v, i: losses.top_logits(x.long(), 2), TypeError),
    (lambda x, v, i: losses.top_logits(x[:, :0], 1), ValueError),
    (lambda x, v, i: losses.top_logits(x, 2, temperature=0.0), ValueError),
    (lambda x, v, i: losses.top_logits(x, 2, temperature=float("nan")), ValueError),
    (lambda x, v, i: losses.distill_xent(x[0], v, i), ValueError),
    (lambda x, v, i: losses.distill_xent(x, v[:2], i[:2]), ValueError),
    (lambda x, v, i: losses.distill_xent(x, v, i[:, :2]), ValueError),
    (lambda x, v, i: losses.distill_xent(x, v[:, :0], i[:, :0]), ValueError),
    (lambda x, v, i: losses.distill_xent(x, v, i.to(torch.int16)), TypeError),
    (lambda x, v, i: losses.distill_xent(x, v.long(), i), TypeError),
    (lambda x, v, i: losses.distill_xent(x, v, i, torch.zeros(2)), ValueError),
    (lambda x, v, i: losses.distill_xent(x, v, i, torch.zeros(3, 1)), ValueError),
    (lambda x, v, i: losses.distill_xent(x, v, i, temperature=-1.0), ValueError),
])
def test_refusals(call, error):
  x = make(3, 20, torch.float32)
  v, i, _ = losses.top_logits(x, 4)
  with pytest.raises(error):
    call(x, v, i)


# ------------------------------------------------------------------------------------- GPU
def check_top(x, k, temperature=1.0):
  v, i, rest = losses.top_logits(x, k, temperature=temperature)
  want_i, want_rest = top_oracle(x, k, temperature)
  assert v.dtype == x.dtype and i.dtype == torch.int32 and rest.dtype == torch.float32
  assert torch.equal(i.cpu(), want_i)
  bits = torch.int32 if x.dtype == torch.float32 else torch.int16  # torch's own gather rewrites NaN
  assert torch.equal(v.cpu().view(bits), x.cpu().contiguous().view(bits).gather(1, want_i.long()))
  # `rest` is fp32: the lowest fp32 value over a temperature below 1 lies outside its range (-inf).
  torch.testing.assert_close(rest.cpu().double(), want_rest.float().double(), rtol=F32, atol=F32,
                             equal_nan=True)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,n,k,pad", [
    (1, 1, 1, 0), (3, 2, 2, 1), (2, 7, 3, 0), (5, 9, 9, 4), (4, 64, 10, 0), (3, 257, 256, 0),
    (2, 1000, 20, 0), (7, 1001, 17, 7), (2, 5003, 256, 0), (300, 4097, 33, 0), (1, 21843, 64, 5),
    (2, 70001, 200, 0)])
def test_top_logits_kernel(dtype, rows, n, k, pad):
  check_top(make(rows, n, dtype, pad=pad, device="cuda"), k, 2.0)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_top_logits_kernel_of_rows_with_ties_masks_and_infinities(dtype):
  n = 6007
  low = torch.finfo(dtype).min
  x = make(12, n, dtype, device="cuda")
  x[0] = 1.5                         # all equal: the lowest classes
  x[1] = -math.inf                   # nothing left by the mask
  x[2] = low
  x[3] = -math.inf
  x[3, 4000:4003] = 2.0              # fewer finite values than k
  x[4] = low
  x[4, 17::301] = 1.0
  x[5, 100] = math.nan
  x[5, 200] = math.inf
  x[6, 50:90] = math.inf             # more infinities than k
  x[7] = x[7].round()                # many ties
  x[8] = 0.0
  x[8, 1::2] = -0.0                  # equal zeros
  x[9, 5] = 60000.0 if dtype == torch.float16 else 1e6  # the others far below
  x[10] = -5.0
  x[10, 3000:] = -6.0
  x[11, ::2] = -math.inf
  for k in (1, 20, 256):
    check_top(x, k)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,k", [(257, 171), (300, 200), (700, 256), (1000, 120), (1001, 200), (2049, 250),
                                 (3001, 171), (6001, 256)])
def test_top_logits_kernel_of_many_kept_in_few_vectors(dtype, n, k):
  low = torch.finfo(dtype).min
  x = make(9, n, dtype, device="cuda")
  x[0] = 1.5
  x[1] = -math.inf
  x[1, n // 2:n // 2 + 40] = 2.0     # fewer finite values than k
  x[2, 3:] = low
  x[3] = x[3].round()
  x[4, 7::2] = math.nan
  x[5, : k - 1] = math.inf
  x[6, ::2] = -math.inf
  x[7] = torch.where(x[7] > 0, torch.zeros_like(x[7]), -torch.zeros_like(x[7]))
  check_top(x, k, 0.7)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [9, 12, 40, 300])
def test_top_logits_kernel_of_negative_rows_with_lowest_masks(dtype, n):
  # Bounds between the largest values and the masks' value are no elements, and huge.
  for cut in (1, 2, 3, 7):
    x = -make(10, n, dtype, seed=cut, pad=7, device="cuda").abs()
    x[:, cut:] = torch.finfo(dtype).min
    for k in (1, 2, 5):
      check_top(x, k, 2.0)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_top_logits_kernel_of_wide_rows_with_ties(dtype):
  n = 50021  # several CTAs share a row
  x = make(3, n, dtype, device="cuda")
  x[0] = 0.25
  x[1] = -math.inf
  x[1, n - 5:] = 3.0
  x[2] = (x[2] * 2).round()
  check_top(x, 100, 0.5)


@gpu
def test_top_logits_kernel_strides_and_offsets():
  base = make(6, 400, torch.bfloat16, device="cuda")
  check_top(base[:, 3:390], 12)       # rows that start inside a vector
  check_top(base[::2, 1:], 5)
  check_top(base.t()[:350], 4)        # transposed
  check_top(base[0].expand(4, 400), 3)
  v, i, rest = losses.top_logits(base[:0], 3)
  assert v.shape == (0, 3) and i.shape == (0, 3) and rest.shape == (0,)


def check_distill(x, values, indices, rest, temperature=1.0, dloss=None):
  rows, n = x.shape
  x = x.detach().requires_grad_()
  if dloss is None:
    dloss = torch.linspace(0.5, 1.5, rows, device=x.device)
  loss = losses.distill_xent(x, values, indices, rest, temperature=temperature)
  (grad,) = torch.autograd.grad(loss, x, dloss)
  want, want_grad = distill_oracle(x, values, indices, rest, temperature, dloss)
  assert loss.dtype == torch.float32 and grad.dtype == x.dtype and grad.shape == x.shape
  torch.testing.assert_close(loss.cpu().double(), want, rtol=F32, atol=F32)
  # q - p of probabilities that are each off by F32 relative; fp16 rounds below 2^-14 absolutely.
  scale = temperature * dloss.abs().cpu().double()[:, None]
  tiny = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
  far = (grad.cpu().double() - want_grad).abs()
  assert bool((far <= 2 * F32 * scale + HALF_STEP[x.dtype] * want_grad.abs() + tiny).all()), far.max()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("with_rest", [False, True])
@pytest.mark.parametrize("rows,n,k,pad", [
    (1, 2, 1, 0), (3, 5, 5, 3), (2, 9, 4, 0), (5, 100, 10, 4), (4, 1000, 20, 0), (3, 1003, 300, 5),
    (320, 515, 7, 0), (2, 21843, 64, 5), (2, 60007, 30, 0)])
def test_distill_kernel(dtype, with_rest, rows, n, k, pad):
  x = make(rows, n, dtype, pad=pad, device="cuda")
  t = make(rows, n, dtype, seed=3, device="cuda")
  values, order = t.float().sort(dim=1, descending=True)
  rest = torch.logsumexp(values[:, k:] / 2.0, 1) if with_rest else None
  check_distill(x, values[:, :k].to(dtype), order[:, :k].to(torch.int32), rest, 2.0)


@gpu
@pytest.mark.parametrize("with_rest", [False, True])
def test_distill_kernel_entries_that_do_not_count(with_rest):
  x = make(6, 777, torch.bfloat16, device="cuda")
  t = teacher_of(x, 9, 1.0)
  idx = t.indices.long()
  idx[0, 5:] = -1
  idx[1, 2] = 777                    # outside
  idx[1, 3] = 1 << 40
  idx[2, 6] = idx[2, 1]              # listed twice
  idx[2, 8] = idx[2, 1]
  idx[3] = -1                        # nothing kept
  idx[4, :] = idx[4, 0]
  values = t.values.cuda()
  values[5, 4] = -math.inf
  rest = t.rest.cuda() if with_rest else None
  check_distill(x, values, idx.cuda(), rest)


@gpu
@pytest.mark.parametrize("n", [700, 40009])
def test_distill_kernel_masked_logits(n):
  for mask in (-math.inf, torch.finfo(torch.float32).min):
    x = make(4, n, torch.float32, device="cuda")
    t = make(4, n, torch.float32, seed=5, device="cuda")
    x[0, 11::2] = mask
    t[0, 11::2] = mask
    x[1, 20:] = mask                  # few classes left
    t[1, 20:] = mask
    x[2, 5:] = mask
    t[2, 5:] = mask
    values, idx, rest = losses.top_logits(t, 16)
    if mask == -math.inf:
      check_distill(x, values, idx, rest)
    else:  # the oracle's softmax of -3e38 / T needs no special case
      check_distill(x, values, idx, rest, 0.7)
  x = torch.full((2, n), torch.finfo(torch.float32).min, device="cuda")
  check_distill(x, torch.zeros(2, 3, device="cuda"), torch.tensor([[1, 2, 3]] * 2, device="cuda"), None)


@gpu
def test_distill_kernel_far_apart_and_equal():
  x = make(4, 300, torch.float32, device="cuda")
  x[0, 3] = 90.0                      # everything else underflows
  x[1] *= 20
  t = teacher_of(x, 5, 1.0)
  check_distill(x, t.values.cuda(), t.indices.cuda(), t.rest.cuda())
  same = losses.top_logits(x, 5, temperature=4.0)
  loss = losses.distill_xent(x, *same, temperature=4.0)
  assert float(loss.abs().max()) < 16 * F32 * F32 * 10 + 1e-8


@gpu
def test_distill_rows_with_zero_weight_are_not_read():
  x = make(5, 999, torch.bfloat16, device="cuda", pad=1)
  v, i, rest = losses.top_logits(make(5, 999, torch.bfloat16, seed=2, device="cuda"), 8)
  x[3] = math.nan
  x = x.requires_grad_()
  w = torch.tensor([1.0, 0.0, 0.5, 0.0, 1.0], device="cuda")
  loss = losses.distill_xent(x, v, i, rest)
  (g,) = torch.autograd.grad(loss, x, w, retain_graph=True)
  assert bool((g[[1, 3]] == 0).all()) and bool((g[[0, 2, 4]] != 0).any(1).all())
  assert math.isnan(float(loss[3].detach())) and bool(torch.isfinite(loss[[0, 1, 2, 4]]).all())
  (g2,) = torch.autograd.grad(loss, x, w)  # a second backward pass of the same graph
  assert torch.equal(g, g2)
  # The gradient's padding columns (what a padded head's backward GEMM may load) are zero.
  assert g.stride(0) % 8 == 0


@gpu
def test_distill_expanded_gradient_and_layouts():
  x = make(33, 130, torch.float16, device="cuda")
  v, i, rest = losses.top_logits(make(33, 130, torch.float16, seed=2, device="cuda"), 6)
  xg = x.detach().requires_grad_()
  losses.distill_xent(xg, v, i, rest).mean().backward()  # expanded d_loss
  want = distill_oracle(x, v, i, rest, 1.0, torch.full((33,), 1 / 33))[1]
  far = (xg.grad.cpu().double() - want).abs()
  assert bool((far <= 2 * F32 + 2.0 ** -11 * want.abs() + 2.0 ** -25).all())
  check_distill(x[:, 3:], v, i - 3, rest)                        # rows inside vectors, index -1
  check_distill(x.t()[:100], v[:1].expand(100, 6), i[:1].expand(100, 6) % 33, None)
  wide = torch.stack([v, v], 2)[:, :, 0]                         # values with a column stride
  check_distill(x, wide, i.long(), rest)
  empty = losses.distill_xent(x[:0].requires_grad_(), v[:0], i[:0], rest[:0])
  assert empty.shape == (0,)
  (g,) = torch.autograd.grad(empty.sum(), [xg], allow_unused=True)
  assert g is None


@gpu
def test_distill_side_stream_and_graph_replay():
  x = make(64, 3001, torch.bfloat16, device="cuda")
  y = make(64, 3001, torch.bfloat16, seed=9, device="cuda")
  teacher = make(64, 3001, torch.bfloat16, seed=4, device="cuda")

  def step(xx):
    xx = xx.detach().requires_grad_()
    top = losses.top_logits(teacher, 32, temperature=2.0)
    loss = losses.distill_xent(xx, *top, temperature=2.0)
    (g,) = torch.autograd.grad(loss, xx, torch.ones_like(loss))
    return loss.detach(), g

  want_x, want_y = step(x), step(y)
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    got = step(x)
  torch.cuda.current_stream().wait_stream(side)
  assert all(torch.equal(a, b) for a, b in zip(got, want_x))
  buf = x.clone()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    step(buf)
  torch.cuda.current_stream().wait_stream(side)
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    out = step(buf)
  for src, want in ((y, want_y), (x, want_x)):
    buf.copy_(src)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, want))


@gpu
@pytest.mark.parametrize("n,k", [(21843, 64), (50021, 200), (900, 256)])
def test_results_do_not_depend_on_the_run(n, k):
  x = make(64, n, torch.bfloat16, device="cuda")
  y = make(64, n, torch.bfloat16, seed=8, device="cuda").requires_grad_()

  def step():
    top = losses.top_logits(x, k)
    loss = losses.distill_xent(y, *top)
    return (*top, loss.detach(), *torch.autograd.grad(loss.sum(), y))

  first = step()
  for _ in range(5):
    assert all(torch.equal(a, b) for a, b in zip(first, step()))


@gpu
def test_second_derivatives_are_refused():
  x = make(3, 50, torch.float32, device="cuda").requires_grad_()
  top = losses.top_logits(make(3, 50, torch.float32, seed=4, device="cuda"), 5)
  (grad,) = torch.autograd.grad(losses.distill_xent(x, *top).sum(), x, create_graph=True)
  with pytest.raises(RuntimeError):
    grad.sum().backward()


@gpu
def test_offsets_past_32_bits():
  """The last rows of logits with more than 2^31 elements."""
  n, few, copies = 21843, 500, 200
  block = make(few, n, torch.bfloat16, device="cuda")
  x = block.repeat(copies, 1)
  assert x.numel() > 2 ** 31
  small, large = losses.top_logits(block, 20), losses.top_logits(x, 20)
  for part in (slice(None, few), slice(-few, None)):
    assert torch.equal(small.values, large.values[part])
    assert torch.equal(small.indices, large.indices[part])
    # 500 * 21843 * 199 elements further on a row starts elsewhere within 16 bytes: other vectors, so
    # its fp32 sum is added in another order.
    torch.testing.assert_close(small.rest, large.rest[part], rtol=F32, atol=F32)
  # Loss and gradient: rows of one CTA in both calls, so that both add in the same order.
  block, x = block[:, :2000].contiguous(), None
  wide = torch.empty(few * copies, n, dtype=torch.bfloat16, device="cuda")[:, :2000]
  wide.copy_(block.repeat(copies, 1))
  teacher = losses.top_logits(block.flip(1).contiguous(), 20)
  found = []
  for logits, times in ((block, 1), (wide, copies)):
    logits = logits.detach().requires_grad_()
    loss = losses.distill_xent(logits, *(t.repeat(times, *[1] * (t.dim() - 1)) for t in teacher))
    (grad,) = torch.autograd.grad(loss, logits, torch.ones_like(loss))
    found.append((loss.detach()[-few:], grad[-few:]))
  # fp32 sums of 2000 exponentials in another split, and one rounding of the gradient to bf16.
  torch.testing.assert_close(found[1][0], found[0][0], rtol=1e-4, atol=1e-4)
  torch.testing.assert_close(found[1][1].float(), found[0][1].float(), rtol=2.0 ** -7, atol=1e-6)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [1e5, 1e7, 1e10, 1e13, 1e20, 3e30])
def test_distill_kernel_of_huge_logits(dtype, size):
  n, k = 700, 6
  x = (make(6, n, dtype, device="cuda") * size).clone()
  x[1] = -x[1].abs()
  x[2, ::2] = -size
  x[3] = size
  x[4] = -size
  x[5, 10:] = -math.inf
  values, indices, rest = losses.top_logits(make(6, n, dtype, seed=2, device="cuda"), k)
  x[0, indices[0].long()] += size
  for keep_rest in (True, False):
    z = x.clone().requires_grad_()
    loss = losses.distill_xent(z, values, indices, rest if keep_rest else None)
    (grad,) = torch.autograd.grad(loss.sum(), z)
    want, want_grad = distill_oracle(x, values, indices, rest if keep_rest else None, 1.0,
                                     torch.ones(6))
    # The loss is fp32: half a step of it, besides fp32 sums of 700 exponentials.
    torch.testing.assert_close(loss.detach().cpu().double(), want.float().double(), rtol=1e-5, atol=1e-4)
    # Gradients lie in [-1, 1]: fp32 sums, one rounding to the type, and the anchor's (2^-24 of |x| c is
    # taken back, what a product x c itself rounds is not larger than the last bit of the difference).
    torch.testing.assert_close(grad.cpu().double(), want_grad, rtol=2.0 ** -7 if dtype == torch.bfloat16 else 1e-4,
                               atol=1e-4)
