"""The two opt-in uses of 8-bit rows in the engine: training with 8-bit activation checkpoints (CLIMB_AMD_ACT8=1, ViltEngine.act8) and evaluation with int8
linear products (CLIMB_AMD_EVAL_I8=1, ViltEngine.eval_i8), against the same model without them."""
import os

import numpy as np
import pytest
import torch

from oracle import vilt_oracle as vo
from tests.test_gpu_parity import enc_to_inputs, grads_of, make_model

pytestmark = pytest.mark.gpu
H16 = os.environ.get("CLIMB_AMD_H16", "bf16")


def _model(**flags):
    model, _ = make_model(["vqa"], 42, precision=H16)
    eng = model._host.engine()
    for k, v in flags.items():
        setattr(eng, k, v)
    return model, eng


def _batch(B, seed):
    enc = vo.synthetic_encodings(B, seed=seed, ragged_text=True)
    return (*enc_to_inputs(enc), vo.synthetic_vqa_targets(B, seed=seed))


def _rel(a, b):
    return float((a.double() - b.double()).norm() / (b.double().norm() + 1e-30))


def _tensors(o, seen, depth=0):
    if isinstance(o, torch.Tensor):
        seen[o.untyped_storage().data_ptr()] = o.untyped_storage().nbytes()
    elif isinstance(o, (list, tuple)):
        for v in o:
            _tensors(v, seen, depth + 1)
    elif isinstance(o, dict):
        for v in o.values():
            _tensors(v, seen, depth + 1)
    elif hasattr(o, "buf"):
        _tensors(o.buf, seen, depth + 1)
    return seen


@pytest.fixture(scope="module")
def steps():
    """one training step of the same model and batch: plain 16-bit, with checkpoints, and the fp32 mode"""
    images, texts, target = _batch(5, 3)
    out = {}
    for name in ("plain", "act8", "fp32"):
        if name == "fp32":
            if H16 == "fp16":
                continue          # (one process, one 16-bit type; the fp32 mode needs neither)
            model, _ = make_model(["vqa"], 42, precision="fp32")
        else:
            model, eng = _model(act8=name == "act8")
        model.train()
        loss, (pooled, logits), _, _ = model.fused_forward_backward("vqa", images, texts, target)
        out[name] = (float(loss), pooled.cpu(), logits.cpu(), grads_of(model))
        if name != "fp32":
            ws = vars(eng.last_ws)
            kept = ("ck", "qkv", "ctx") if name == "act8" else ("x", "h1", "xn", "hn", "u", "a", "qkv", "ctx")
            out[name + "_bytes"] = sum(_tensors([ws[k] for k in kept], {}).values())
    return out


def test_checkpointed_step_has_the_plain_steps_gradients(steps):
    """The forward differs from the plain one in one rounding (the GELU reads its input in 16 bits), so loss and outputs agree to the 16-bit mode's own noise.
    The backward reads activations whose codes err by at most half a step of max / 63.5 of 64 values (normal data: 2.5 sigma / 63.5 / sqrt 12 = 1.1 % r.m.s.): a
    weight gradient inherits that once, a layer's input gradient through LayerNorm and GELU' about as much again, and 12 layers add independent errors to a
    residual stream that carries most of the gradient past them: 1.1 % (1 + sqrt(12) / 2) = 3 % expected, 8 % allowed; a checkpoint read with a wrong scale,
    layout, layer or statistic is off by far more."""
    loss, pooled, logits, G = steps["act8"]
    l0, p0, o0, G0 = steps["plain"]
    assert abs(loss - l0) < 2e-3 * abs(l0) and _rel(pooled, p0) < 0.03 and _rel(logits, o0) < 0.03
    assert set(G) == set(G0)
    worst = ("", 0.0)
    for n in G0:
        if n.endswith("attention.key.bias"):          # identically zero up to rounding
            continue
        r = _rel(G[n], G0[n])
        worst = max(worst, (n, r), key=lambda t: t[1])
        assert r < 0.08, (n, r)
    print("worst gradient:", worst)
    if "fp32" in steps:          # ... and is hardly further from the fp32 mode than the plain 16-bit step
        Gf = steps["fp32"][3]
        a = float(np.median([_rel(G[n], Gf[n]) for n in Gf if not n.endswith("key.bias")]))
        b = float(np.median([_rel(G0[n], Gf[n]) for n in Gf if not n.endswith("key.bias")]))
        print("median error against fp32: checkpoints %.4f, plain %.4f" % (a, b))
        assert a < b + 0.03


def test_checkpoints_take_less_than_half_of_the_saved_activations(steps):
    """a layer keeps 6 H (q, k, v) + 2 H (attention output) + 8 H (codes; 1 / 64 more of exponents) bytes a token instead of 36 H"""
    print("bytes kept:", steps["plain_bytes"], "->", steps["act8_bytes"])
    M, H = 5 * 192, 768
    assert steps["plain_bytes"] >= 12 * M * H * 36 and steps["act8_bytes"] < 0.47 * steps["plain_bytes"]


def test_checkpointed_step_beside_other_work():
    """a forward without gradients between a training forward and its backward; two backwards into one gradient; the captured step.  Two runs of one step are not
    the same bits (the heads' products split their sums with atomics), and a last bit that moves there moves 16-bit roundings below it by a step, 2^-7 of
    single elements: 2 % of a gradient's norm is allowed.  Another batch's activations, a stale checkpoint or a sum taken twice is of order 1."""
    same = 0.02
    model, eng = _model(act8=True)
    images, texts, target = _batch(3, 7)
    other = _batch(3, 8)
    model.train()
    crit = torch.nn.BCEWithLogitsLoss(reduction="mean")

    def backward(between):
        model.zero_grad(set_to_none=True)
        _, logits = model("vqa", images, texts)
        if between:
            with torch.no_grad():
                model("vqa", other[0], other[1])
        (crit(logits, target.to(logits.device).float()) * target.shape[1]).backward()
        return grads_of(model)
    a, b = backward(False), backward(True)
    for n in a:
        assert _rel(b[n], a[n]) < same or n.endswith("key.bias"), n
    model.zero_grad(set_to_none=True)
    model.fused_forward_backward("vqa", images, texts, target)
    one = grads_of(model)
    model.fused_forward_backward("vqa", images, texts, target)
    two = grads_of(model)
    for n in one:
        assert _rel(two[n], 2 * one[n]) < same or n.endswith("key.bias"), n
    model.zero_grad(set_to_none=True)
    for seed in (7, 9, 7):
        im, tx, tg = _batch(3, seed)
        model.zero_grad(set_to_none=True)
        want = model.fused_forward_backward("vqa", im, tx, tg)[0]
        gw = grads_of(model)
        model.zero_grad(set_to_none=True)
        got = model.graphed_forward_backward("vqa", im, tx, tg)[0]
        gg = grads_of(model)
        assert abs(float(got) - float(want)) <= 1e-5 * abs(float(want))
        for n in gw:
            assert _rel(gg[n], gw[n]) < same or n.endswith("key.bias"), n


def test_frozen_layers_and_optimizer_with_checkpoints():
    model, eng = _model(act8=True)
    for n, p in model.named_parameters():
        if ".embeddings." in n or any(f"encoder.layer.{i}." in n for i in range(9)):
            p.requires_grad = False
    images, texts, target = _batch(2, 11)
    model.train()
    opt = model.create_optimizer(dict(lr=1e-4, weight_decay=1e-2, adam_epsilon=1e-8)) if False else None
    model.fused_forward_backward("vqa", images, texts, target)
    G = grads_of(model)
    assert not any("encoder.layer.8." in n for n in G) and any("encoder.layer.9." in n for n in G)
    ref, _ = _model()
    for n, p in ref.named_parameters():
        p.requires_grad = not (".embeddings." in n or any(f"encoder.layer.{i}." in n for i in range(9)))
    ref.train()
    ref.fused_forward_backward("vqa", images, texts, target)
    R = grads_of(ref)
    assert set(R) == set(G)
    for n in R:
        if not n.endswith("key.bias"):
            assert _rel(G[n], R[n]) < 0.08, n


def test_act8_refuses_what_it_does_not_cover():
    model, eng = _model(act8=True)
    eng.cls_only_last = True
    images, texts, target = _batch(2, 1)
    with pytest.raises(NotImplementedError, match="act8"):
        model.fused_forward_backward("vqa", images, texts, target)


def test_8_bit_rows_go_with_the_16_bit_types():
    if H16 == "fp16":
        pytest.skip("one process, one 16-bit type")
    images, texts, target = _batch(2, 1)
    for flag in ("act8", "eval_i8"):
        model, _ = make_model(["vqa"], 42, precision="fp32")
        setattr(model._host.engine(), flag, True)
        with pytest.raises(NotImplementedError, match="16-bit"):
            model.fused_forward_backward("vqa", images, texts, target)


def test_a_forward_that_raised_leaves_no_trace(monkeypatch):
    """an evaluation that ends in the middle of the encoder: the next training step is the plain one"""
    images, texts, target = _batch(3, 2)
    plain, _ = _model()
    model, eng = _model(eval_i8=True)
    attn = type(eng).attn_fwd
    def fail(*a, **k):
        raise KeyboardInterrupt
    monkeypatch.setattr(type(eng), "attn_fwd", fail)
    with pytest.raises(KeyboardInterrupt):
        _evaluate(model, images, texts)
    monkeypatch.setattr(type(eng), "attn_fwd", attn)
    for m in (plain, model):
        m.train()
    a, b = (m.fused_forward_backward("vqa", images, texts, target) for m in (plain, model))
    assert abs(float(a[0]) - float(b[0])) < 1e-5 * abs(float(a[0]))
    p, _ = _evaluate(model, images, texts)
    fresh, _ = _model(eval_i8=True)
    want, _ = _evaluate(fresh, images, texts)
    assert _rel(p, want) < 1e-5


def _evaluate(model, images, texts):
    model.eval()
    with torch.no_grad():
        pooled, logits = model("vqa", images, texts)
    return pooled.cpu(), logits.cpu()


def test_int8_evaluation():
    """tokens and weights in int8: 0.7 % r.m.s. an operand (3 sigma / 127 / sqrt 12), 1 % a product, 48 products of which each adds to a residual stream: a few
    per cent of the outputs; 10 % allowed"""
    images, texts, _ = _batch(6, 5)
    plain, _ = _model()
    model, eng = _model(eval_i8=True)
    p0, o0 = _evaluate(plain, images, texts)
    eng.prof = {"kernel": "linear_i8", "events": []}
    p1, o1 = _evaluate(model, images, texts)
    assert len(eng.prof["events"]) == 48          # four products a layer went through the int8 kernels
    eng.prof = None
    print("int8 evaluation: pooled %.4f logits %.4f" % (_rel(p1, p0), _rel(o1, o0)))
    assert 0 < _rel(p1, p0) < 0.1 and _rel(o1, o0) < 0.1
    # training forwards are untouched, and the codes follow the parameters
    target = vo.synthetic_vqa_targets(6, seed=5)
    for m in (plain, model):
        m.train()
        m.zero_grad(set_to_none=True)
    a = plain.fused_forward_backward("vqa", images, texts, target)
    b = model.fused_forward_backward("vqa", images, texts, target)
    assert abs(float(a[0]) - float(b[0])) < 1e-5 * abs(float(a[0]))
    with torch.no_grad():
        for n, p in model.named_parameters():
            if n.endswith("output.dense.weight") or n.endswith("query.weight"):
                p.mul_(1.5)
    p2, _ = _evaluate(model, images, texts)
    fresh, _ = _model(eval_i8=True)
    fresh.load_state_dict(model.state_dict())
    p3, _ = _evaluate(fresh, images, texts)
    assert _rel(p2, p1) > 0.05 and _rel(p2, p3) < 1e-5


def test_int8_evaluation_after_an_optimizer_step():
    """FusedAdamW writes the parameters through the C ABI: the next evaluation multiplies by the new ones"""
    images, texts, target = _batch(4, 6)
    model, eng = _model(eval_i8=True)
    opt = model.create_optimizer({"lr": 1e-2, "weight_decay": 0.0, "adam_epsilon": 1e-8})
    before, _ = _evaluate(model, images, texts)
    model.train()
    model.fused_forward_backward("vqa", images, texts, target)
    opt.step()
    opt.zero_grad()
    after, _ = _evaluate(model, images, texts)
    fresh, _ = _model(eval_i8=True)
    fresh.load_state_dict(model.state_dict())
    want, _ = _evaluate(fresh, images, texts)
    assert _rel(after, want) < 1e-5 and _rel(after, before) > 1e-3


@pytest.mark.parametrize("first", [True, False])
def test_act8_switched_between_forward_and_backward(first):
    """the backward reads what its forward kept, whatever the switch says by then (an even batch: the rows that the deferred weight gradients take)"""
    images, texts, target = _batch(4, 13)
    crit = torch.nn.BCEWithLogitsLoss(reduction="mean")
    out = []
    for switch in (False, True):
        model, eng = _model(act8=first)
        model.train()
        _, logits = model("vqa", images, texts)
        if switch:
            eng.act8 = not first
        (crit(logits, target.to(logits.device).float()) * target.shape[1]).backward()
        out.append(grads_of(model))
    assert set(out[0]) == set(out[1])
    for n in out[0]:
        assert _rel(out[1][n], out[0][n]) < 0.02 or n.endswith("key.bias"), n          # (0.02: two runs' last bits, as above)


def test_forwards_without_gradients_hold_no_checkpoints():
    """act8 keeps memory down: an evaluation's workspace -- of its own batch size, or beside a pending backward -- has neither checkpoints nor the backward's scratch"""
    model, eng = _model(act8=True)
    images, texts, target = _batch(3, 17)
    other = _batch(5, 18)
    p0, _ = _evaluate(model, other[0], other[1])
    names = ("ck", "part8", "wg8", "du_a")
    assert [w for w in eng._ws.values()] and not any(getattr(w, n, None) is not None for w in eng._ws.values() for n in names)
    model.train()
    crit = torch.nn.BCEWithLogitsLoss(reduction="mean")
    _, logits = model("vqa", images, texts)
    with torch.no_grad():
        model("vqa", images, texts)
    assert sorted(getattr(w, "ck", None) is not None for w in eng._ws.values()) == [False, False, True]
    (crit(logits, target.to(logits.device).float()) * target.shape[1]).backward()
    G = grads_of(model)
    plain, _ = _model()
    assert _rel(p0, _evaluate(plain, other[0], other[1])[0]) < 1e-2
    plain.train()
    _, logits = plain("vqa", images, texts)
    (crit(logits, target.to(logits.device).float()) * target.shape[1]).backward()
    for n, r in grads_of(plain).items():
        assert n.endswith("key.bias") or _rel(G[n], r) < 0.08, n


@pytest.mark.parametrize("eager_first", [True, False])
def test_int8_evaluation_captured(eager_first):
    """a captured evaluation, with or without an eager one before it: replays beside eager work and after parameter updates (through torch and through the fused
    optimizer) multiply by the parameters of their time, and so do the eager evaluations after a capture"""
    images, texts, target = _batch(4, 21)
    other = _batch(4, 22)
    model, eng = _model(eval_i8=True)
    model.eval()
    opt = model.create_optimizer({"lr": 1e-2, "weight_decay": 0.0, "adam_epsilon": 1e-8})
    eng.refresh_shadow()          # (what the 16-bit parts of the forward read)
    im, tx = images.cuda(), {k: v.cuda() for k, v in texts.items()}
    if eager_first:
        _evaluate(model, images, texts)
    eng.eval_i8 = False          # (the first run of everything else: workspaces, LDS limits)
    _evaluate(model, im, tx)
    eng.eval_i8 = True
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g), torch.no_grad():
        pooled, logits = model("vqa", im, tx)

    def fresh(i, t):
        m, _ = _model(eval_i8=True)
        m.load_state_dict(model.state_dict())
        return _evaluate(m, i, t)[0]
    first = None
    for step in range(3):
        for i, t in ((images, texts), (other[0], other[1])):
            want = fresh(i, t)
            im.copy_(i)
            for k in tx:
                tx[k].copy_(t[k])
            g.replay()
            torch.cuda.synchronize()
            assert _rel(pooled.cpu(), want) < 1e-5, step
            if first is None:
                first = want
            assert _rel(_evaluate(model, i, t)[0], want) < 1e-5, step
        if step == 0:
            with torch.no_grad():
                for n, p in model.named_parameters():
                    if n.endswith("output.dense.weight") or n.endswith("query.weight"):
                        p.mul_(1.5)
        else:
            model.train()
            model.fused_forward_backward("vqa", images, texts, target)
            opt.step()
            opt.zero_grad()
            model.eval()
    assert _rel(fresh(images, texts), first) > 1e-3


def _ewc(model, P):
    import types
    from climb_amd.cl_algorithms import EWC
    from tests.test_gpu_parity import _ewc_state
    ewc = EWC(types.SimpleNamespace(ewc_fisher_sample_percentage=0.01, ewc_loss_weight=100.0))
    ewc.set_task_state("nlvr2", model, *_ewc_state(P, 5))
    return ewc


@pytest.mark.parametrize("config", ["plain", "frozen9", "ewc", "accumulate"])
def test_training_steps_with_checkpoints_and_the_optimizer(config):
    """two steps with the optimizer named (its promise to run next holds weight-gradient launches back in the plain mode; with checkpoints there are none to hold):
    after the first the moments are the gradients, so they agree as gradients do (8 %, as above; the EWC term is fp32 in both); all 16-bit shadows are the images
    of the fp32 parameters; the second step's loss, through those shadows, agrees to 2 % -- a step of AdamW moves a weight by lr whatever its gradient's size, and
    where 3 % of noise turns a gradient's sign the two models move apart by 2 lr of it"""
    import random
    res = {}
    for name in ("plain", "act8"):
        torch.manual_seed(0)
        random.seed(0)
        model, P = make_model(["vqa", "nlvr2"], 42, precision=H16)
        eng = model._host.engine()
        eng.act8 = name == "act8"
        model.train()
        if config == "frozen9":
            model.get_encoder().freeze_bottom_k_layers(9)
        ewc = _ewc(model, P) if config == "ewc" else None
        opt = model.create_optimizer({"lr": 2e-5, "weight_decay": 1e-2, "adam_epsilon": 1e-8})
        opt.zero_grad()
        names, orig = [], eng._timed_call

        def spy(kernel, flops, call, *a, _o=orig, _l=names):
            _l.append(call)
            return _o(kernel, flops, call, *a)
        eng._timed_call = spy
        losses, extra, m1 = [], [], None
        for step in range(2):
            images, texts, target = _batch(4, 30 + step)
            if config == "accumulate" and step == 0:
                model.fused_forward_backward("vqa", images, texts, target, ewc, optimizer=opt)
            loss, _, _, el = model.fused_forward_backward("vqa", images, texts, target, ewc, optimizer=opt)
            opt.step()
            opt.zero_grad()
            assert not bool(eng.grad.any())
            losses.append(float(loss))
            extra.append(float(el) if el is not None else 0.0)
            if m1 is None:
                m1 = {n: opt._m[eng.layout.offset[n]:eng.layout.offset[n] + eng.layout.numel(n)].cpu() for n in eng.layout.shapes}
        eng.refresh_shadow()
        torch.cuda.synchronize()
        t16 = eng.t16
        assert torch.equal(eng._shadow, eng.flat.to(t16))
        for n, N, K in eng._linear_weight_names():
            o, ot = eng.layout.offset[n], eng._t_off[n]
            assert torch.equal(eng._shadow_t[ot:ot + N * K].view(K, N), eng._shadow[o:o + N * K].view(N, K).t()), n
        assert bool(torch.isfinite(eng.flat).all()) and bool((opt._v >= 0).all())
        grouped = [n for n in names if "grouped" in n]
        assert not grouped if name == "act8" else grouped, grouped
        assert ("climb_act8_weight_grad" in names) == (name == "act8")
        res[name] = (losses, extra, m1)
        del model, opt, eng
    (l0, e0, m0), (l1, e1, m1) = res["plain"], res["act8"]
    for a, b in zip(l0, l1):
        assert abs(a - b) <= 2e-2 * abs(a), (l0, l1)
    for a, b in zip(e0, e1):
        assert abs(a - b) <= 1e-3 * max(1.0, abs(a)), (e0, e1)
    moved = [n for n in m0 if bool(m0[n].any())]
    assert moved == [n for n in m1 if bool(m1[n].any())] and any("layer.11" in n for n in moved)
    assert any("layer.8." in n for n in moved) == (config != "frozen9")
    for n in moved:
        assert n.endswith("key.bias") or _rel(m1[n], m0[n]) < 0.08, (n, _rel(m1[n], m0[n]))


def _two_modes(make, run):
    """gradients of one step of the same model without and with checkpoints"""
    out = []
    for on in (False, True):
        model = make()
        model._host.engine().act8 = on
        out.append(run(model) + (grads_of(model),))
        del model
    return out


@pytest.mark.parametrize("task", ["nlvr2", "vcr"])
def test_checkpointed_steps_of_tasks_with_several_images_or_choices(task):
    """two images an example (two sequences, one joint head) and four choices (four sequences); 8 % as above"""
    b, n = 3, dict(nlvr2=2, vcr=4)[task]
    e = vo.synthetic_encodings(n * b, seed=41, ragged_text=True)
    if task == "nlvr2":
        images, texts = e["pixel_values"], {k: e[k][:b] for k in ("input_ids", "token_type_ids", "attention_mask")}
    else:
        images, texts = e["pixel_values"][:b], {k: e[k] for k in ("input_ids", "token_type_ids", "attention_mask")}
    labels = torch.tensor([1, 0, 1])

    def run(model):
        model.eval()          # (no dropout mask in the choices' head)
        loss, (pooled, logits), _, _ = model.fused_forward_backward(task, images, texts, labels)
        return float(loss), logits.cpu()
    (l0, o0, G0), (l1, o1, G1) = _two_modes(lambda: make_model([task], 42, precision=H16)[0], run)
    assert abs(l1 - l0) < 2e-2 * abs(l0) and _rel(o1, o0) < 0.05 and set(G0) == set(G1)
    for k in G0:
        if k == "task_layer.vcr.1.bias":          # one number added to all choices of a softmax: its gradient is the sum of (p - y) over them, 1 - 1 = 0 up to rounding
            assert float(G0[k].abs().max()) < 1e-6 and float(G1[k].abs().max()) < 1e-6
            continue
        assert k.endswith("key.bias") or _rel(G1[k], G0[k]) < 0.08, (k, _rel(G1[k], G0[k]))


def test_checkpointed_step_of_vilt_on_bert_features():
    """the embeddings come from a frozen text encoder: their gradient ends at LayerNorm's input; 8 % as above"""
    from oracle import bert_oracle as bo
    from climb_amd.modeling import create_continual_learner_map
    from climb_amd.configs.task_configs import task_configs
    from climb_amd.configs.model_configs import model_configs
    P, PB = vo.init_params(["vqa"], 42), bo.init_bert_params(7)
    sd = {k.replace("vilt_encoder.", "viltbert_encoder."): v for k, v in P.items()}
    sd.update({"viltbert_encoder.bert." + k: v for k, v in PB.items()})
    images, texts, target = _batch(4, 43)

    def make():
        model = create_continual_learner_map["viltbert"](model_name_or_path="random-init:0", ordered_cl_tasks=["vqa"], model_config=model_configs["viltbert"],
                                                         task_configs=task_configs, device=torch.device("cuda:0"), precision=H16)
        model.load_state_dict(sd, strict=True)
        return model.to(torch.device("cuda:0"))

    def run(model):
        model.eval()          # (no dropout masks in the text encoder)
        loss, (pooled, logits), _, _ = model.fused_forward_backward("vqa", images, texts, target)
        return float(loss), logits.cpu()
    (l0, o0, G0), (l1, o1, G1) = _two_modes(make, run)
    assert abs(l1 - l0) < 2e-3 * abs(l0) and _rel(o1, o0) < 0.05 and set(G0) == set(G1) and not any("word_embeddings" in k or ".bert." in k for k in G1)
    for k in G0:
        assert k.endswith("key.bias") or _rel(G1[k], G0[k]) < 0.08, (k, _rel(G1[k], G0[k]))


def test_ranges_reported_by_a_checkpointed_backward_are_final():
    """what a data-parallel reducer hooks: every range of the gradient buffer is reported once, and holds by then what it holds at the end; the groups are those of
    the plain mode (ranks may run different paths, but have to issue the same collectives)"""
    images, texts, target = _batch(4, 47)
    seen = {}
    for name in ("plain", "act8"):
        model, eng = _model(act8=name == "act8")
        model.train()
        model.fused_forward_backward("vqa", images, texts, target)          # (workspaces)
        model.zero_grad(set_to_none=True)
        reports = []
        eng.grad_ready_hook = lambda lo, hi: reports.append((lo, hi, eng.grad[lo:hi].clone()))
        model.fused_forward_backward("vqa", images, texts, target)
        eng.grad_ready_hook = None
        torch.cuda.synchronize()
        for lo, hi, g in reports:
            assert torch.equal(g, eng.grad[lo:hi]), (name, lo, hi)
        spans = sorted((lo, hi) for lo, hi, _ in reports)
        assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:]))
        seen[name] = [(lo, hi) for lo, hi, _ in reports]
        assert bool(eng.grad.any())
    assert seen["plain"] == seen["act8"] and len(seen["act8"]) >= 4


def test_int8_evaluation_under_an_active_adapter():
    """the base's products in int8, the adapter's bottleneck in 16 bits; 10 % allowed as without one"""
    import types
    from climb_amd.cl_algorithms import AdapterHandler
    images, texts, _ = _batch(5, 51)
    out = []
    for on in (False, True):
        model, _ = make_model(["vqa", "nlvr2"], 42, precision=H16)
        handler = AdapterHandler("vanilla", types.SimpleNamespace(adapter_config="houlsby", adapter_reduction_factor=16, ordered_cl_tasks=["vqa", "nlvr2"]))
        handler.add_adapters_to_model(model)
        g = torch.Generator().manual_seed(7)
        with torch.no_grad():
            for n, p in model.named_parameters():
                if ".adapters." in n:
                    p.copy_((torch.randn(p.shape, generator=g) * (0.05 if n.endswith("weight") else 0.02)).to(p.device))
        handler.activate_adapter_for_eval("vqa", model)
        eng = model._host.engine()
        eng.eval_i8 = on
        names, orig = [], eng._timed_call

        def spy(kernel, flops, call, *a, _o=orig, _l=names):
            _l.append(call)
            return _o(kernel, flops, call, *a)
        eng._timed_call = spy
        p, o = _evaluate(model, images, texts)
        out.append((p, o))
        assert names.count("climb_linear_i8") == (48 if on else 0)
        handler.activate_adapter_for_eval("nlvr2", model)
        q, _ = _evaluate(model, images, texts)
        assert _rel(q, p) > 0.05          # another adapter, another function
    print("int8 evaluation under an adapter: pooled %.4f logits %.4f" % (_rel(out[1][0], out[0][0]), _rel(out[1][1], out[0][1])))
    assert 0 < _rel(out[1][0], out[0][0]) < 0.1 and _rel(out[1][1], out[0][1]) < 0.1


def test_both_uses_in_one_model():
    """int8 evaluations in the checkpointed training's workspace (activations in buffers that the layers share), between a training forward and its backward and after"""
    images, texts, target = _batch(4, 61)
    crit = torch.nn.BCEWithLogitsLoss(reduction="mean")
    only, _ = _model(eval_i8=True)
    want, _ = _evaluate(only, images, texts)
    ck, _ = _model(act8=True)
    ck.train()
    _, logits = ck("vqa", images, texts)
    (crit(logits, target.to(logits.device).float()) * target.shape[1]).backward()
    G = grads_of(ck)
    model, eng = _model(act8=True, eval_i8=True)
    assert _rel(_evaluate(model, images, texts)[0], want) < 1e-5
    model.train()
    _, logits = model("vqa", images, texts)
    assert _rel(_evaluate(model, images, texts)[0], want) < 1e-5
    model.train()
    (crit(logits, target.to(logits.device).float()) * target.shape[1]).backward()
    for n, g in grads_of(model).items():
        assert _rel(g, G[n]) < 0.02 or n.endswith("key.bias"), n          # (0.02: two runs' last bits, as above)
    assert _rel(_evaluate(model, images, texts)[0], want) < 1e-5
