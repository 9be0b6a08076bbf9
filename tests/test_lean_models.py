"""The lean training steps (8-bit checkpoints, the head's loss without logits) next to the ordinary ones
of the same parameters."""
import pytest
import torch

from vodascheduler_amd.models import BertBase, TransformerNMT, get_workload, prepare_model
from vodascheduler_amd.models.layers import EncoderLayer, FeedForward
from vodascheduler_amd.ops.act8 import Act8Linear
from vodascheduler_amd.ops.xent import softmax_cross_entropy


def _bert(act8, seed=0):
    torch.manual_seed(seed)
    return BertBase(vocab=500, seq_len=24, d_model=64, heads=2, d_ff=160, layers=2, act8=act8)


def _bert_batch(dev, B=6, T=24, P=5):
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(1, 500, (B, T), generator=g)
    mask = torch.ones(B, T, dtype=torch.bool)
    mask[:, -4:] = False
    pos = torch.argsort(torch.rand(B, T - 4, generator=g), 1)[:, :P]
    labels = torch.gather(ids, 1, pos)
    labels[0, :2] = -100
    return [t.to(dev) for t in (ids, mask, pos, labels)]


def _step(model, batch, lean):
    ids, mask, pos, labels = batch
    if lean:
        loss, correct, n = model.head_metrics(ids, mask, pos, labels)
    else:
        loss, correct, n = softmax_cross_entropy(model(ids, mask, pos), labels.reshape(-1), model.num_classes)
    loss.backward()
    return float(loss.detach()), int(correct), int(n), {k: p.grad.float().clone() for k, p in model.named_parameters()}


def _rel(a, b):
    return float((a - b).norm() / b.norm().clamp_min(1e-12))


def _compare(dev, dtype):
    plain, lean = _bert(False), _bert(True)
    lean.load_state_dict(plain.state_dict())
    plain, lean = plain.to(dev, dtype), lean.to(dev, dtype)
    batch = _bert_batch(dev)
    lp, cp, np_, gp = _step(plain, batch, False)
    ll, cl, nl, gl = _step(lean, batch, True)
    assert nl == np_ == 28
    # the forward is the same function: the loss differs by the activations' own roundings
    tol = 0.02 if dtype == torch.bfloat16 else 1e-5
    assert abs(ll - lp) < tol * lp and (dtype == torch.bfloat16 or cl == cp)
    for k, g in gp.items():
        if float(g.norm()) < 1e-6:
            continue  # key biases: their gradient is zero, what is left is rounding
        # weights next to a checkpoint see inputs to within e4m3's 2^-4 a value, 2^-4 in any norm; what
        # flows back through two GELUs sees their slopes at those inputs
        assert _rel(gl[k], g) < (0.14 if dtype == torch.bfloat16 else 2 * 2.0 ** -4), (k, _rel(gl[k], g))


def test_bert_step_on_the_cpu():
    _compare(torch.device("cpu"), torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_bert_step_on_the_gpu(dtype):
    _compare(torch.device("cuda", 0), dtype)


def test_translation_head():
    torch.manual_seed(0)
    m = TransformerNMT(vocab=300, seq_len=8, d_model=32, d_ff=64, heads=2, key_dim=16)
    src, tgt = torch.randint(1, 300, (4, 8)), torch.randint(1, 300, (4, 9))
    tgt[1, 5:] = 0
    want = softmax_cross_entropy(m(src, tgt[:, :-1]).reshape(-1, 300), tgt[:, 1:].reshape(-1), 300, 0)
    got = m.head_metrics(src, tgt[:, :-1], tgt[:, 1:])
    for g, w in zip(got, want):
        torch.testing.assert_close(g.detach().double(), w.detach().double())


def test_feed_forward_parameters_and_refusal():
    a, b = FeedForward(16, 32, "gelu"), FeedForward(16, 32, "gelu", act8=True)
    b.load_state_dict(a.state_dict())
    x = torch.randn(3, 16)
    torch.testing.assert_close(a(x), b(x))
    assert isinstance(b.fc1, Act8Linear) and b.fc2.act == "gelu"
    with pytest.raises(ValueError):
        FeedForward(16, 32, "relu", act8=True)


@pytest.mark.gpu
@pytest.mark.parametrize("amp", [True, False])
@pytest.mark.parametrize("name", ["bert-base-lean", "transformer-lean"])
def test_workload_trains_on_the_trainer_s_path(name, amp, monkeypatch):
    """bf16 weights under autocast (or fp32), flat gradients, the fused optimizer, the engine's readiness
    hooks: one step runs, every parameter gets a finite gradient, and the flat gradients agree with a
    step of the ordinary workload."""
    from vodascheduler_amd.ops.optim import make_optimizer
    from vodascheduler_amd.parallel.comm import LocalCommunicator
    from vodascheduler_amd.parallel.ddp import ElasticDDP
    from vodascheduler_amd.utils.flat import grad_of

    dev = torch.device("cuda", 0)

    def step(workload):
        w = get_workload(workload)
        torch.manual_seed(0)
        m = prepare_model(w, dev, amp=amp).train()
        opt = make_optimizer(w.optimizer, m.parameters(), **{**w.opt_kwargs, "lr": 0.0})
        ddp = ElasticDDP(m, LocalCommunicator(dev), opt)
        batch = w.make_batch(8, dev, torch.Generator(device=dev).manual_seed(1))
        for _ in range(2):  # the second step after the engine's calibration
            opt.zero_grad()
            with torch.autocast("cuda", dtype=torch.bfloat16, enabled=amp, cache_enabled=False):
                loss, correct, n = w.metrics(m, batch)
            loss.backward()
            ddp.finalize()
        torch.cuda.synchronize()
        return float(loss.detach()), int(n), {k: grad_of(p).float().clone() for k, p in m.named_parameters()}

    lean, plain = step(name), step(name.removesuffix("-lean"))
    assert lean[1] == plain[1] and abs(lean[0] - plain[0]) < (0.02 if amp else 1e-4) * plain[0]
    for k, g in plain[2].items():
        assert torch.isfinite(lean[2][k]).all(), k
        if "head" in k or "mlm_out.bias" in k:
            assert _rel(lean[2][k], g) < (0.03 if amp else 1e-4), (k, _rel(lean[2][k], g))


@pytest.mark.gpu
def test_a_layer_keeps_less():
    """What one BERT layer keeps for the backward: at least a third less with act8."""
    from vodascheduler_amd.models import cast_compute_weights_

    kept = {}
    for act8 in (False, True):
        torch.manual_seed(0)
        m = cast_compute_weights_(EncoderLayer(256, 4, 1024, act="gelu", act8=act8).cuda()).train()
        x = torch.randn(64, 128, 256, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        with torch.autocast("cuda", dtype=torch.bfloat16, cache_enabled=False):
            y = m(x)
        torch.cuda.synchronize()
        kept[act8] = torch.cuda.memory_allocated() - before
        y.float().sum().backward()
        del y, x, m
    assert kept[True] < 0.67 * kept[False], kept
