"""Workloads of the gated MLP and of the distillation operators, with their plain forms.

Operators:

* ``vmoe_b200.ops.expert_gated_mlp``: ``y = (act(x Wg^T + bg) * (x Wu^T + bu)) Wo^T + bo`` per
  expert, forward (serving) and forward + backward (training).
* ``vmoe_b200.ops.losses.top_logits``: a teacher's ``k`` largest logits per example, sorted, and
  the log-sum-exp of all the others.
* ``vmoe_b200.ops.losses.distill_xent``: the divergence of a student from such a teacher, per
  example, and its gradient.

``run`` computes them with elementary fp32 operations while ``own`` is false and through the
package's entry points once it is true.
"""
import math

import torch

own = False

_DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


def listed():
  return [
      # One image's class token after the last block, ViT-B width: latency of a single row.
      dict(name="gated_one_row", op="gated", train=False, e=1, r=1, h=768, m=2048, act="gelu",
           bias=True, residual=True),
      # The pooled probes of 13 images in an attention-pooling head of ViT-H width.
      dict(name="gated_pooled_rows", op="gated", train=False, e=1, r=13, h=1280, m=5120,
           act="silu", bias=True, residual=False),
      # Eight experts serving one image: 197 tokens, two experts each, a few rows per expert.
      dict(name="gated_few_rows_experts", op="gated", train=False, e=8, r=52, h=1024, m=2736,
           act="silu", bias=False, residual=False),
      # A batch of 32 images at 384 pixels (577 tokens) through a dense block, evaluation.
      dict(name="gated_dense_eval", op="gated", train=False, e=1, r=18464, h=1024, m=2736,
           act="gelu", bias=True, residual=True),
      # A small fine-tuning batch with ragged rows: 5 images of 257 tokens, ViT-H width.
      dict(name="gated_dense_train_small", op="gated", train=True, e=1, r=1285, h=1280, m=3416,
           act="silu", bias=True, residual=False),
      # The experts of one block in pre-training: 128 images, capacity ratio 1.05.
      dict(name="gated_experts_train", op="gated", train=True, e=8, r=6620, h=768, m=2048,
           act="gelu", bias=True, residual=False),
      # Ten best of one served example, ImageNet-1k classes.
      dict(name="top_one_example", op="top", rows=1, n=1000, k=10, dtype="float32", pad=0,
           temperature=1.0),
      # A few examples over a large label space (text vocabulary), many kept.
      dict(name="top_wide", op="top", rows=24, n=131101, k=200, dtype="bfloat16", pad=0,
           temperature=2.0),
      # The teacher's answer to a pre-training batch, ImageNet-21k classes, rows padded to a
      # multiple of 8 as the classification head writes them.
      dict(name="top_batch", op="top", rows=4096, n=21843, k=64, dtype="bfloat16", pad=5,
           temperature=2.0),
      # A micro-step over ImageNet-1k classes with fp32 logits.
      dict(name="distill_small", op="distill", rows=96, n=1000, k=20, dtype="float32", pad=0,
           temperature=1.0, rest=True),
      # Few examples, a wide label space, kept classes renormalised.
      dict(name="distill_wide", op="distill", rows=37, n=131101, k=100, dtype="float16", pad=0,
           temperature=3.0, rest=False),
      # A pre-training batch over ImageNet-21k classes.
      dict(name="distill_batch", op="distill", rows=4096, n=21843, k=64, dtype="bfloat16", pad=5,
           temperature=2.0, rest=True),
  ]


def _log_between(rng, low, high):
  return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
  op = rng.choice(["gated", "gated", "top", "distill"])
  if op == "gated":
    train = rng.random() < 0.5
    most = 18 * 8 * 6620 * 768 * 2048  # the largest listed case
    while True:
      e = rng.choice([1, 1, 1, 2, 4, 8, 16])
      r = _log_between(rng, 1, 16384 // e)
      h = 8 * _log_between(rng, 24, 160)
      m = 8 * _log_between(rng, 48, 640)
      if 3 * (6 if train else 2) * e * r * h * m <= most and e * h * m <= 1 << 25:
        break
    return dict(op="gated", train=train, e=e, r=r, h=h, m=m, act=rng.choice(["gelu", "silu"]),
                bias=rng.random() < 0.5, residual=rng.random() < 0.5)
  n = _log_between(rng, 100, 131101)
  rows = _log_between(rng, 1, max(1, min(4096, 4096 * 21843 // n)))
  case = dict(op=op, rows=rows, n=n, k=min(n, _log_between(rng, 1, 256)),
              dtype=rng.choice(["bfloat16", "bfloat16", "float16", "float32"]),
              pad=rng.choice([0, -n % 8]), temperature=rng.choice([1.0, 2.0, 4.0]))
  if case["dtype"] == "float32":
    case["rows"] = max(1, rows // 2)
  if op == "distill":
    case["rest"] = rng.random() < 0.5 and case["k"] < n
  return case


def _logits(gen, rows, n, pad, dtype):
  """Logits as a classification head leaves them: a per-example scale, a few strong classes."""
  dev = gen.device
  base = torch.randn(rows, n + pad, generator=gen, device=dev)
  base.mul_(1.0 + torch.rand(rows, 1, generator=gen, device=dev))
  strong = torch.randint(0, n, (rows, min(n, 12)), generator=gen, device=dev)
  base.scatter_add_(1, strong, 6 * torch.rand(strong.shape, generator=gen, device=dev))
  return base.to(dtype)[:, :n]


def prepare(case, seed):
  gen = torch.Generator(device="cuda")
  gen.manual_seed(seed)
  dev = gen.device
  s = dict(case)
  if case["op"] == "gated":
    e, r, h, m = (case[k] for k in ("e", "r", "h", "m"))

    def rand(*shape, scale=1.0):
      return (torch.randn(*shape, generator=gen, device=dev) * scale).to(torch.bfloat16)

    s["x"] = rand(e, r, h)
    if e > 1 and r > 16:
      s["x"][:, r - r // 16:] = 0  # the empty slots at the end of an expert's buffer
    s["w_in"] = rand(e, 2, m, h, scale=(2.0 / (h + m)) ** 0.5 * 1.5)
    s["w_out"] = rand(e, h, m, scale=(2.0 / (h + m)) ** 0.5)
    s["b_in"] = rand(e, 2, m, scale=0.1) if case["bias"] else None
    s["b_out"] = rand(e, h, scale=0.1) if case["bias"] else None
    s["res"] = rand(e, r, h) if case["residual"] else None
    s["dy"] = rand(e, r, h) if case["train"] else None
    if case["train"]:
      for k in ("x", "w_in", "w_out", "b_in", "b_out", "res"):
        if s[k] is not None:
          s[k].requires_grad_()
    return s
  rows, n, k, t = case["rows"], case["n"], case["k"], case["temperature"]
  dtype = _DTYPES[case["dtype"]]
  s["logits"] = _logits(gen, rows, n, case["pad"], dtype)
  if case["op"] == "distill":
    teacher = (0.5 * s["logits"].float() + 0.7 * _logits(gen, rows, n, 0, torch.float32)).to(dtype)
    values, indices = teacher.float().topk(k, dim=1)
    others = (teacher.float() / t).scatter(1, indices, -math.inf)
    if k > 2:  # a few examples whose teacher kept fewer classes
      fewer = torch.rand(rows, 1, generator=gen, device=dev) < 0.05
      place = torch.arange(k, device=dev)
      drop = fewer & (place >= k // 2)
      others.scatter_(1, indices, torch.where(drop, values / t, torch.full_like(values, -math.inf)))
      indices = torch.where(drop, torch.full_like(indices, -1), indices)
    s["values"] = values.to(dtype)
    s["indices"] = indices.to(torch.int32)
    s["others"] = torch.logsumexp(others, dim=1) if case["rest"] else None
    # fp16 gradients carry a loss scale, or the far classes' would underflow.
    s["weight"] = torch.rand(rows, generator=gen, device=dev) * \
        (4096.0 if dtype == torch.float16 else 1.0 / rows)
    if rows > 8:
      s["weight"][-(rows // 16 + 1):] = 0  # the padding examples of the last batch
    s["logits"].requires_grad_()
  return s


# ------------------------------------------------------------------------------- plain forms
def _sigmoid(x):
  return 1.0 / (1.0 + torch.exp(-x))


def _gate_and_slope(g, act):
  """The activation and its derivative."""
  if act == "silu":
    sg = _sigmoid(g)
    return g * sg, sg * (1.0 + g * (1.0 - sg))
  c = math.sqrt(2.0 / math.pi)
  t = torch.tanh(c * (g + 0.044715 * g * g * g))
  slope = 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * g * g)
  return 0.5 * g * (1.0 + t), slope


def _plain_gated(s):
  with torch.no_grad():
    f = {k: None if s[k] is None else s[k].float()
         for k in ("x", "w_in", "w_out", "b_in", "b_out", "res", "dy")}
    x, wg, wu, wo = f["x"], f["w_in"][:, 0], f["w_in"][:, 1], f["w_out"]
    g, u = torch.bmm(x, wg.transpose(1, 2)), torch.bmm(x, wu.transpose(1, 2))
    if f["b_in"] is not None:
      g, u = g + f["b_in"][:, 0:1], u + f["b_in"][:, 1:2]
    a, slope = _gate_and_slope(g, s["act"])
    hid = a * u
    y = torch.bmm(hid, wo.transpose(1, 2))
    if f["b_out"] is not None:
      y = y + f["b_out"][:, None]
    if f["res"] is not None:
      y = y + f["res"]
    out = {"y": y.bfloat16()}
    if s["train"]:
      dy = f["dy"]
      dhid = torch.bmm(dy, wo)
      dg, du = dhid * u * slope, dhid * a
      out["dx"] = (torch.bmm(dg, wg) + torch.bmm(du, wu)).bfloat16()
      out["dw_in"] = torch.stack([torch.bmm(dg.transpose(1, 2), x),
                                  torch.bmm(du.transpose(1, 2), x)], dim=1).bfloat16()
      out["dw_out"] = torch.bmm(dy.transpose(1, 2), hid).bfloat16()
      if f["b_in"] is not None:
        out["db_in"] = torch.stack([dg.sum(1), du.sum(1)], dim=1).bfloat16()
        out["db_out"] = dy.sum(1).bfloat16()
      if f["res"] is not None:
        out["dres"] = s["dy"]
    return out


def _lse(x):
  top = x.amax(dim=1, keepdim=True)
  top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
  return torch.log(torch.exp(x - top).sum(dim=1)) + top[:, 0]


def _plain_top(s):
  x = s["logits"].float()
  order = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :s["k"]]
  rest = (x / s["temperature"]).scatter(1, order, -math.inf)
  return {"values": s["logits"].gather(1, order), "indices": order.int(), "rest": _lse(rest)}


def _plain_distill(s):
  # Exponentials of all classes in 32 bits; their sums and the terms of the kept classes, whose
  # first-order parts cancel where student and teacher agree, in 64.
  with torch.no_grad():
    t = s["temperature"]
    valid = s["indices"] >= 0
    at = s["indices"].long().clamp(min=0)
    z = s["logits"].float() / t
    top = z.amax(dim=1, keepdim=True)
    ez = torch.exp(z - top)
    kept = torch.zeros_like(z, dtype=torch.bool).scatter_add(1, at, valid)
    rest_sum = ez.masked_fill(kept, 0.0).sum(dim=1, dtype=torch.float64)
    zk = s["logits"].gather(1, at).double() / t - top
    all_s = torch.log(rest_sum + (torch.exp(zk) * valid).sum(1))
    v = (s["values"].double() / t).masked_fill(~valid, -math.inf)
    if s["others"] is not None:
      v = torch.cat([v, s["others"].double()[:, None]], dim=1)
    log_p = v - _lse(v)[:, None]
    log_q = zk - all_s[:, None]
    if s["others"] is not None:
      log_q = torch.cat([log_q, (torch.log(rest_sum) - all_s)[:, None]], dim=1)
    p = torch.exp(log_p)
    loss = torch.where(p > 0, p * (log_p - log_q), torch.zeros_like(p)).sum(1)
    k = at.shape[1]
    slope = (torch.exp(log_q[:, :k]) - p[:, :k]) * valid
    outside = 1.0 - torch.exp(log_p[:, k:] - log_q[:, k:]) if s["others"] is not None \
        else torch.ones_like(p[:, :1])
    q = torch.exp(z - top - all_s[:, None].float()) * outside.float()
    q = q.masked_fill(kept, 0.0).scatter_add(1, at, slope.float())
    dlogits = q * (t * s["weight"])[:, None]
    return {"loss": (loss * t * t).float(), "dlogits": dlogits.to(s["logits"].dtype)}


# ------------------------------------------------------------------------------- the operators
def _own_gated(s):
  from vmoe_b200 import ops
  y = ops.expert_gated_mlp(s["x"], s["w_in"], s["b_in"], s["w_out"], s["b_out"], act=s["act"],
                           residual=s["res"])
  out = {"y": y}
  if s["train"]:
    names = [k for k in ("x", "w_in", "w_out", "b_in", "b_out", "res") if s[k] is not None]
    grads = torch.autograd.grad(y, [s[k] for k in names], s["dy"])
    out.update(("d" + k, g) for k, g in zip(names, grads))
    out["y"] = y.detach()
  return out


def _own_top(s):
  from vmoe_b200.ops import losses
  values, indices, rest = losses.top_logits(s["logits"], s["k"], temperature=s["temperature"])
  return {"values": values, "indices": indices, "rest": rest}


def _own_distill(s):
  from vmoe_b200.ops import losses
  loss = losses.distill_xent(s["logits"], s["values"], s["indices"], s["others"],
                             temperature=s["temperature"])
  (dlogits,) = torch.autograd.grad(loss, [s["logits"]], s["weight"])
  return {"loss": loss.detach(), "dlogits": dlogits}


def run(s):
  if own:
    return {"gated": _own_gated, "top": _own_top, "distill": _own_distill}[s["op"]](s)
  return {"gated": _plain_gated, "top": _plain_top, "distill": _plain_distill}[s["op"]](s)


def work(case):
  if case["op"] == "gated":
    e, r, h, m = (case[k] for k in ("e", "r", "h", "m"))
    weights = 3 * e * m * h + (e * (2 * m + h) if case["bias"] else 0)
    rows = e * r * h
    size = weights + rows * (3 if case["residual"] else 2)
    flops = 6 * e * r * h * m
    if case["train"]:
      size += weights + rows * (3 if case["residual"] else 2)
      flops *= 3
    return {"bytes": 2 * size, "flops": flops}
  rows, n, k = case["rows"], case["n"], case["k"]
  width = 4 if case["dtype"] == "float32" else 2
  if case["op"] == "top":
    return {"bytes": rows * (n * width + k * (width + 4) + 4), "flops": 3 * rows * n}
  size = rows * (2 * n * width + k * (width + 4) + 8 + (4 if case["rest"] else 0))
  return {"bytes": size, "flops": 6 * rows * n}


# ------------------------------------------------------------------------------- 64 bits
def _exact_gated(s):
  names = [k for k in ("x", "w_in", "w_out", "b_in", "b_out", "res") if s[k] is not None]
  d = {k: s[k].detach().double().requires_grad_(bool(s["train"])) for k in names}
  pre = torch.einsum("erh,ecmh->cerm", d["x"], d["w_in"])
  if "b_in" in d:
    pre = pre + d["b_in"].permute(1, 0, 2)[:, :, None]
  fn = torch.nn.functional
  gate = fn.silu(pre[0]) if s["act"] == "silu" else fn.gelu(pre[0], approximate="tanh")
  y = torch.einsum("erm,ehm->erh", gate * pre[1], d["w_out"])
  if "b_out" in d:
    y = y + d["b_out"].unsqueeze(1)
  if "res" in d:
    y = y + d["res"]
  out = {"y": y.detach()}
  if s["train"]:
    grads = torch.autograd.grad(y, [d[k] for k in names], s["dy"].double())
    out.update(("d" + k, g) for k, g in zip(names, grads))
  return out


def _exact_top(s):
  x = s["logits"].double()
  ordered = x.sort(dim=1, descending=True)[0]
  rest = torch.logsumexp(ordered[:, s["k"]:] / s["temperature"], dim=1) \
      if s["k"] < s["n"] else torch.full((s["rows"],), -math.inf, device=x.device)
  return {"values": ordered[:, :s["k"]].clone(), "indices": None, "rest": rest.double()}


def _exact_distill(s):
  t, n = s["temperature"], s["n"]
  x = s["logits"].detach().double().requires_grad_()
  log_q = torch.log_softmax(x / t, dim=1)
  # Kept classes and "any other class" as one distribution of n + 1 outcomes.
  at = torch.where(s["indices"] < 0, n + 1, s["indices"]).long()
  target = torch.full((s["rows"], n + 2), -math.inf, dtype=torch.float64, device=x.device)
  target.scatter_(1, at, s["values"].double() / t)
  is_kept = torch.zeros_like(target).scatter_(1, at, 1.0)[:, :n] > 0
  target = target[:, :n + 1]
  if s["others"] is not None:
    target[:, n] = s["others"].double()
  log_p = torch.log_softmax(target, dim=1)
  p = log_p.exp()
  entropy = torch.where(p > 0, p * log_p, torch.zeros_like(p)).sum(1)
  cross = (p[:, :n] * log_q).sum(1)
  if s["others"] is not None:
    cross = cross + p[:, n] * torch.logsumexp(log_q.masked_fill(is_kept, -math.inf), dim=1)
  loss = t * t * (entropy - cross)
  (dlogits,) = torch.autograd.grad(loss, [x], s["weight"].double())
  return {"loss": loss.detach(), "dlogits": dlogits}


def exact(case, seed):
  s = prepare(case, seed)
  return {"gated": _exact_gated, "top": _exact_top, "distill": _exact_distill}[case["op"]](s)
