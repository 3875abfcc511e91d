"""Gated MLP blocks in the models, distillation in the trainer, and the two together."""
import copy
import os

import pytest
import torch

from vmoe_b200 import ops
from vmoe_b200.checkpoints import flax_layout
from vmoe_b200.models import naming, vit_moe, vit_moe_ensemble
from vmoe_b200.ops import losses
from vmoe_b200.parallel import mesh as mesh_lib
from vmoe_b200.train import trainer
from vmoe_b200.utils import misc
from vmoe_b200.utils.config_dict import ConfigDict

gpu = pytest.mark.gpu
STEP = 2.0 ** -8  # half a step of bf16, relative to the value


def model_config(gate="silu", classifier="gap", **encoder):
  return {
      "num_classes": 5, "patch_size": (8, 8), "hidden_size": 16, "image_size": 16,
      "classifier": classifier, "representation_size": None,
      "encoder": {"num_layers": 2, "num_heads": 2, "mlp_dim": 24, "dropout_rate": 0.0,
                  "attention_dropout_rate": 0.0, "mlp_gate": gate,
                  "moe": {"num_experts": 2, "layers": (1,), "group_size": 8,
                          "router": {"num_selected_experts": 1, "noise_std": 0.0,
                                     "dispatcher": {"name": "einsum", "capacity": 8,
                                                    "batch_priority": False}}}, **encoder}}


def build(seed=0, **kwargs):
  torch.manual_seed(seed)
  return vit_moe.VisionTransformerMoe(**model_config(**kwargs))


# --------------------------------------------------------------------------------- models
def test_parameters_in_the_checkpoint_layout():
  model = build(classifier="map")
  shapes = {k: tuple(v[0]) for k, v in
            misc.flatten_dict(flax_layout.flax_shapes(model), sep="/").items()}
  dense, moe = "Encoder/encoderblock_0/Mlp/", "Encoder/encoderblock_1/Moe/Mlp/"
  for prefix, experts in ((dense, ()), (moe, (2,))):
    got = {k[len(prefix):]: v for k, v in shapes.items() if k.startswith(prefix)}
    assert got == {"Dense_gate/kernel": experts + (16, 24), "Dense_gate/bias": experts + (24,),
                   "Dense_up/kernel": experts + (16, 24), "Dense_up/bias": experts + (24,),
                   "Dense_out/kernel": experts + (24, 16), "Dense_out/bias": experts + (16,)}
  assert sum(k.endswith("Dense_up/kernel") for k in shapes) == 3  # dense, experts, pooling head
  assert sum(int(torch.tensor(s).prod()) for s in shapes.values()) == sum(
      p.numel() for p in model.parameters())
  keys = [k for k, _, _ in naming.named_flax_parameters(model, prefix="")]
  assert len(set(keys)) == len(keys) and any(k.endswith("Moe/Mlp/Dense_gate/kernel") for k in keys)


def test_checkpoint_round_trip():
  a, b = build(1), build(2)
  tree, specs = flax_layout.to_flax(a)
  leaf = tree["Encoder"]["encoderblock_1"]["Moe"]["Mlp"]["Dense_up"]["kernel"]
  experts = [m for m in a.modules() if isinstance(m, vit_moe.GatedExpertMlp)][0]
  assert torch.equal(torch.as_tensor(leaf), experts.w_in.data[:, 1].transpose(1, 2))
  flax_layout.from_flax(b, tree)
  for (n, p), (_, q) in zip(a.named_parameters(), b.named_parameters()):
    assert torch.equal(p, q), n


@pytest.mark.parametrize("gate", ["gelu", "silu"])
def test_blocks_compute_the_gated_mlp(gate):
  torch.manual_seed(0)
  block = vit_moe.GatedMlpBlock(12, 20, out_dim=8, gate=gate)
  experts = vit_moe.GatedExpertMlp(3, 12, 20, gate=gate, split_rngs=True)
  assert not torch.equal(experts.w_in[0], experts.w_in[1])
  act = torch.nn.functional.silu if gate == "silu" else (
      lambda v: torch.nn.functional.gelu(v, approximate="tanh"))

  def plain(x, m, i):
    x = x.double()
    g = x @ m.w_in[i, 0].double().t() + m.b_in[i, 0].double()
    u = x @ m.w_in[i, 1].double().t() + m.b_in[i, 1].double()
    return (act(g) * u) @ m.w_out[i].double().t() + m.b_out[i].double()

  x, res = torch.randn(2, 5, 12), torch.randn(2, 5, 8)
  # fp32 sums of 12 and 20 products, each off by at most 2^-24 of the magnitudes (below 8 here).
  far = block(x, residual=res).double() - (plain(x, block, 0) + res.double())
  assert far.abs().max() < 36 * 2.0 ** -24 * 8
  x = torch.randn(3, 5, 12)
  far = experts(x).double() - torch.stack([plain(x[i], experts, i) for i in range(3)])
  assert far.abs().max() < 36 * 2.0 ** -24 * 8


def test_dropout_keeps_the_mean_and_is_off_in_inference():
  torch.manual_seed(0)
  block = vit_moe.GatedMlpBlock(8, 16, dropout_rate=0.5)
  x = torch.randn(4, 8)
  still = block.eval()(x)
  assert torch.equal(still, block(x))
  block.train()
  # Output dropout of one half: every entry is 0 or comes from the doubled output.
  y = block(x)
  assert (y == 0).any() and (y != 0).any()
  # Nothing dropped: the composed form is the operator.
  far = vit_moe._gated_with_dropout(x[None], block.w_in, block.b_in, block.w_out, block.b_out,
                                    "gelu", 0.0)[0] - still
  assert far.abs().max() < 30 * 2.0 ** -24 * 8


def test_ensemble_and_mlp_less_settings():
  cfg = model_config()
  cfg["encoder"]["moe"].update(ensemble_size=2, num_experts=4)
  cfg["encoder"]["moe"]["router"].update(num_selected_experts=1)
  cfg["encoder"]["moe"]["router"].pop("dispatcher")
  torch.manual_seed(0)
  model = vit_moe_ensemble.VisionTransformerMoeEnsemble(**cfg)
  assert any(isinstance(m, vit_moe.GatedExpertMlp) for m in model.modules())
  # The experts' setting apart from the dense blocks'.
  model = build(gate=None)
  assert not any(isinstance(m, (vit_moe.GatedMlpBlock, vit_moe.GatedExpertMlp))
                 for m in model.modules())
  cfg = model_config(gate=None)
  cfg["encoder"]["moe"]["mlp_gate"] = "gelu"
  model = vit_moe.VisionTransformerMoe(**cfg)
  assert sum(isinstance(m, vit_moe.GatedExpertMlp) for m in model.modules()) == 1
  assert not any(isinstance(m, vit_moe.GatedMlpBlock) for m in model.modules())
  with pytest.raises(ValueError, match="mlp_gate"):
    build(gate="relu")


def test_cost_of_a_gated_model():
  images = torch.zeros(2, 16, 16, 3)
  plain, gated = (misc.count_forward_flops(build(gate=g), images) for g in (None, "gelu"))
  # One more projection hidden x mlp_dim: 2 images x 4 tokens in the dense block, 2 experts x 8 slots.
  assert gated - plain == 2.0 * 16 * 24 * (8 + 16)


# --------------------------------------------------------------------------------- trainer
def make_state(config, seed=0, device=None, lr=0.1):
  mesh = mesh_lib.get_auto_logical_mesh(1)
  mesh_lib.set_mesh(mesh)
  return trainer.create_train_state(
      model_config={"name": "VisionTransformerMoe", **config}, total_steps=10, mesh=mesh, seed=seed,
      optimizer_config={"name": "sgd", "momentum": 0.0, "learning_rate": lr}, device=device)


def make_batch(n=8, seed=3):
  g = torch.Generator().manual_seed(seed)
  return (torch.randn(n, 16, 16, 3, generator=g),
          torch.nn.functional.one_hot(torch.randint(5, (n,), generator=g), 5).float())


@pytest.mark.parametrize("use_rest", [True, False])
def test_distilled_step_has_the_loss_of_the_formula(use_rest):
  config = model_config()
  state = make_state(config, 0)
  teacher = trainer.create_teacher(model_config={"name": "VisionTransformerMoe", **config}, seed=9)
  assert not teacher.training and not any(p.requires_grad for p in teacher.parameters())
  images, labels = make_batch()
  with torch.no_grad():
    logits = state.model(images)[0].double()
    teacher_logits = teacher(images)[0]
  step = trainer.wrap_train_step_with_distillation(trainer.train_step, teacher, top_k=3,
                                                   temperature=2.0, weight=0.25, use_rest=use_rest)
  before = copy.deepcopy(teacher.state_dict())
  _, metrics = step(state, images, labels, losses.softmax_xent)
  q = torch.softmax(logits / 2, 1)
  p = torch.softmax(teacher_logits.double() / 2, 1)
  top = p.topk(3, 1).indices
  pk, qk = p.gather(1, top), q.gather(1, top)
  if use_rest:
    pk = torch.cat([pk, 1 - pk.sum(1, keepdim=True)], 1)
    qk = torch.cat([qk, 1 - qk.sum(1, keepdim=True)], 1)
  else:
    pk = pk / pk.sum(1, keepdim=True)
  distance = 4 * (pk * (pk.log() - qk.log())).sum(1)
  want = 0.75 * -(labels.double() * torch.log_softmax(logits, 1)).sum(1) + 0.25 * distance
  assert abs(float(metrics["main_loss"]) - float(want.mean())) < 1e-5  # fp32 losses of order 1
  assert all(torch.equal(v, before[k]) for k, v in teacher.state_dict().items())


def test_microsteps_take_the_teachers_rows_of_their_examples():
  config = model_config(moe=None)
  images, labels = make_batch()
  teacher = trainer.create_teacher(model_config={"name": "VisionTransformerMoe", **config}, seed=9)
  step = trainer.wrap_train_step_with_distillation(trainer.train_step, teacher, top_k=2, weight=1.0)
  found = []
  for n in (None, 4):
    state = make_state(config, 0)
    step(state, images, labels, losses.softmax_xent, microsteps=n)
    found.append([p.detach().clone() for p in state.model.parameters()])
  for p, q in zip(*found):
    assert (p - q).abs().max() < 1e-6  # the same mean in another order of fp32 additions


def test_distillation_inside_mixup_and_adversarial_training():
  config = model_config()
  seen = []

  class Teacher(torch.nn.Module):
    def forward(self, images):
      seen.append(images.clone())
      return images.flatten(1)[:, :5]

  state = make_state(config)
  state.rngs["mixup"] = torch.Generator().manual_seed(0)
  images, labels = make_batch()
  student_saw = []

  def train_step(state, images, labels, loss_fn, **kwargs):
    student_saw.append(images.clone())
    return trainer.train_step(state, images, labels, loss_fn, **kwargs)

  step = trainer.wrap_train_step_with_distillation(train_step, Teacher())
  step = trainer.wrap_train_step_with_mixup(step, concentration=1.0)
  _, metrics = step(state, images, labels, losses.softmax_xent)
  assert torch.equal(seen[0], student_saw[0]) and not torch.equal(seen[0], images)
  assert torch.isfinite(metrics["total_loss"])


def test_refusals_of_distillation():
  state = make_state(model_config())
  images, labels = make_batch()
  with pytest.raises(ValueError, match="weight"):
    trainer.wrap_train_step_with_distillation(trainer.train_step, state.model, weight=1.5)
  for classes, rows, match in ((6, 8, "6 classes"), (5, 16, "16 rows")):
    step = trainer.wrap_train_step_with_distillation(
        trainer.train_step, lambda im, c=classes, r=rows: torch.randn(r, c))
    with pytest.raises(ValueError, match=match):
      step(state, images, labels, losses.softmax_xent)


class _Writer:
  def write_scalars(self, step, scalars):
    pass

  write_hparams = write_texts = lambda self, *a: None

  def flush(self):
    pass


def train_config(gate="silu", steps=2, size=16, **extra):
  from vmoe_b200.configs.vmoe_paper import common
  config = common.get_base_config()
  pp = 'value_range(-1,1)|onehot(5, inkey="label", outkey="labels")|keep("image", "labels")'
  data = dict(name="synthetic", batch_size=8, image_size=size, num_classes=5, process=pp)
  config.dataset = ConfigDict(type_safe=False)
  config.dataset.train = ConfigDict(dict(data, split="train", num_train_examples=64,
                                         shuffle_buffer=16), type_safe=False)
  config.dataset.val = ConfigDict(dict(data, split="validation", num_eval_examples=8),
                                  type_safe=False)
  config.train_steps = steps
  config.loss = ConfigDict({"name": "softmax_xent"})
  config.optimizer = ConfigDict({"name": "sgd", "momentum": 0.9, "learning_rate": 0.01},
                                type_safe=False)
  model = model_config(gate)
  model.pop("image_size")
  config.model = ConfigDict({"name": "VisionTransformerMoe", **model}, type_safe=False)
  config.save_checkpoint.every_steps = steps
  config.report_progress.every_steps = 1
  config.evaluate.every_steps = steps
  config.extra_rng_keys = ("dropout", "gating")
  for k, v in extra.items():
    setattr(config, k, v)
  return config


def train_teacher_then_student(tmp_path, dtype, **sizes):
  mesh = mesh_lib.get_auto_logical_mesh(1)
  mesh_lib.set_mesh(mesh)
  first, second = str(tmp_path / "teacher"), str(tmp_path / "student")
  config = train_config(gate=None)
  config.model.encoder.dtype = dtype
  config.model.hidden_size = sizes.get("hidden_size", 16)
  config.model.encoder.mlp_dim = sizes.get("mlp_dim", 24)
  teacher, _ = trainer.train_and_evaluate(config, first, mesh=mesh, writer=_Writer())
  names = sorted(n for n in os.listdir(os.path.join(first, "ckpt")) if "ckpt_2" in n)
  initialization = {"name": "initialize_from_vmoe", "prefix": os.path.join(first, "ckpt", "ckpt_2"),
                    "rules": [("^(params/.*)$", r"\1"), ("^.*$", "")],
                    "raise_if_target_unmatched": False}
  frozen = trainer.create_teacher(model_config=config.model, initialization=initialization,
                                  image_size=16)
  for (n, p), (_, q) in zip(teacher.model.named_parameters(), frozen.named_parameters()):
    assert torch.equal(p.detach().cpu(), q), (n, names)
  student = train_config(
      microsteps=2, mixup=ConfigDict({"concentration": 0.2}, type_safe=False),
      distillation=ConfigDict({"model": config.model, "initialization": initialization,
                               "top_k": 3, "temperature": 2.0, "weight": 0.5}, type_safe=False))
  student.model.encoder.dtype = dtype
  student.model.hidden_size = config.model.hidden_size
  student.model.encoder.mlp_dim = config.model.encoder.mlp_dim
  state, metrics = trainer.train_and_evaluate(student, second, mesh=mesh, writer=_Writer())
  assert state.step == 2 and torch.isfinite(torch.as_tensor(metrics["total_loss"]))


def test_a_gated_student_learns_from_a_saved_teacher(tmp_path):
  train_teacher_then_student(tmp_path, "float32")


# --------------------------------------------------------------------------------- on a GPU
@gpu
def test_a_gated_student_learns_from_a_saved_teacher_on_the_kernels(tmp_path):
  from vmoe_b200.ops import _lib
  _lib.reset_launch_count()
  train_teacher_then_student(tmp_path, "bfloat16", hidden_size=128, mlp_dim=200)
  assert _lib.reset_launch_count() > 50, "the CUDA kernels did not run"


class _Doubled(torch.nn.Module):
  """Expert ``i`` multiplies by ``2^i``: exact, so only the movement of rows can be off."""

  def forward(self, x):
    return x * (2.0 ** torch.arange(x.shape[0], device=x.device)).to(x.dtype)[:, None, None]


@gpu
@pytest.mark.parametrize("items,experts,k,capacity", [(1, 2, 1, 1), (37, 4, 2, 5), (64, 3, 3, 80)])
@pytest.mark.parametrize("residual", [False, True])
def test_rows_of_other_experts_move_on_the_kernels(items, experts, k, capacity, residual):
  """``apply_experts`` with an expert module that is not the plain MLP: dispatch, combine and their
  gradients against the same plan in 64 bits, with full experts, dropped items and empty slots.

  Every output rounds once and the sum of k terms is held in fp32; dx rounds the gate-weighted row
  and the sum: (2^-8 + 2^-8) of the magnitudes; the gates' gradients are fp32 dot products of h
  entries: h * 2^-24 of the magnitudes at most."""
  from vmoe_b200.ops import moe_ops
  g, h = 2, 64
  gen = torch.Generator().manual_seed(7)
  logits = torch.randn(g, items, experts, generator=gen).cuda()
  gates = torch.softmax(logits, -1).requires_grad_()
  x = torch.randn(g, items, h, generator=gen).bfloat16().cuda().requires_grad_()
  res = torch.randn(g, items, h, generator=gen).bfloat16().cuda() if residual else None
  disp = moe_ops.FusedTopKDispatcher(gates, k, capacity, batch_priority=True)
  y = disp.apply_experts(_Doubled(), x, residual=res)
  dy = torch.randn(y.shape, generator=gen).bfloat16().cuda()
  y.backward(dy)
  taken = disp.slot.long() < capacity
  at = disp.expert.long()
  weight = (gates.detach().double().gather(2, at) * taken)
  scale = 2.0 ** at.double()
  xd, dyd = x.detach().double(), dy.double()
  want = (weight * scale).sum(2, keepdim=True) * xd
  bound = 1.1 * STEP * (want + (0 if res is None else res.double())).abs() + 1e-6 * scale.amax()
  want = want if res is None else want + res.double()
  assert bool(((y.detach().double() - want).abs() <= bound).all())
  dx = (weight * scale).sum(2, keepdim=True) * dyd
  assert bool(((x.grad.double() - dx).abs() <= 2.2 * STEP * dx.abs() + 1e-6).all())
  dots = (xd * dyd).sum(2, keepdim=True) * scale * taken
  dgates = torch.zeros_like(gates, dtype=torch.float64).scatter_add(2, at, dots)
  room = h * 2.0 ** -24 * 2 * scale.amax() * (xd * dyd).abs().sum(2, keepdim=True)
  assert bool(((gates.grad.double() - dgates).abs() <= room + 1e-6).all())


def _rounded(t, noise, gen):
  """One rounding to bf16 as its worst half step, in a random direction (``noise`` 0: none)."""
  sign = torch.randint(0, 2, t.shape, generator=gen).double() * 2 - 1
  return t * (1 + noise * STEP * sign)


def _chain_oracle(t, noise, seed):
  """Gated MLP with its residual, head, distillation, in 64 bits: loss and the gradients of x, w_in
  and w_out, with half steps of size ``noise`` at every place where the kernels round."""
  gen = torch.Generator().manual_seed(seed)
  r = lambda v: _rounded(v, noise, gen)
  d = {k: v.detach().cpu().double() for k, v in t.items() if v.is_floating_point()}
  x, (wg, wu), wo = d["x"][0], d["w_in"][0], d["w_out"][0]
  gate = (x @ wg.t()).requires_grad_()
  a = torch.nn.functional.silu(gate)
  (slope,) = torch.autograd.grad(a.sum(), gate)
  a, u = a.detach(), x @ wu.t()
  hid = r(a * u)
  y = r(hid @ wo.t() + x)
  logits = r(y @ d["head"]).requires_grad_()
  loss = losses._distill_reference(logits, d["values"], t["indices"].cpu(), d["rest"], 2.0)
  (dl,) = torch.autograd.grad(loss.double().mean(), logits)
  dy = r(r(dl) @ d["head"].t())
  dh = dy @ wo
  dg, du = r(dh * r(u * slope)), r(dh * r(a))
  return {"loss": loss.detach().double(), "x": r(r(dg @ wg + du @ wu) + dy),
          "w_in": torch.stack([r(dg.t() @ x), r(du.t() @ x)])[None], "w_out": r(dy.t() @ hid)[None]}


@gpu
@pytest.mark.parametrize("rows,h,m,classes,k", [(1, 64, 96, 40, 4), (9, 128, 200, 1001, 16),
                                                (150, 192, 328, 5003, 64)])
def test_teacher_student_loss_and_gradients_in_one_run(rows, h, m, classes, k):
  """Teacher's top logits, gated student, loss, backward as one run, eager and replayed. The bound is the
  oracle's own change when every rounding goes its full half step in a random direction (the largest of
  three draws, times 1.5); actual roundings are a third of that in the mean square."""
  gen = torch.Generator().manual_seed(rows)
  rnd = lambda *s, scale=1.0: (torch.randn(*s, generator=gen) * scale).bfloat16().cuda()
  t = {"x": rnd(1, rows, h), "w_in": rnd(1, 2, m, h, scale=h ** -0.5),
       "w_out": rnd(1, h, m, scale=m ** -0.5), "head": rnd(h, classes, scale=h ** -0.5)}
  teacher = rnd(rows, classes, scale=2.0)

  def step():
    leaves = {n: t[n].detach().requires_grad_() for n in ("x", "w_in", "w_out")}
    top = losses.top_logits(teacher, k, temperature=2.0)
    y = ops.expert_gated_mlp(leaves["x"], leaves["w_in"], None, leaves["w_out"], None, act="silu",
                             residual=leaves["x"])
    loss = losses.distill_xent(y[0] @ t["head"], *top, temperature=2.0)
    return (loss,) + torch.autograd.grad(loss.mean(), list(leaves.values())) + tuple(top)

  def compare(out):
    t.update(values=out[4], indices=out[5], rest=out[6])
    want = _chain_oracle(t, 0.0, 0)
    draws = [_chain_oracle(t, 1.0, s) for s in range(3)]
    for name, got in zip(("loss", "x", "w_in", "w_out"), out):
      room = 1.5 * max(float((d[name] - want[name]).norm()) for d in draws)
      far = float((got.detach().cpu().double().reshape(want[name].shape) - want[name]).norm())
      assert far <= room + 1e-6 * float(want[name].norm()), (name, far, room)

  eager = step()
  compare(eager)
  eager = [v.clone() for v in eager]
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    step()
  torch.cuda.current_stream().wait_stream(side)
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    out = step()
  graph.replay()
  for a, b in zip(out, eager):
    assert torch.equal(a, b)
  teacher.copy_(teacher.flip(0) * 0.5)
  t["x"].copy_(t["x"].flip(1))
  graph.replay()
  compare(out)
