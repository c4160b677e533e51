"""Layer norm, token embedding, top logits and the distillation loss without a GPU: what their entry points refuse, and the
plain statements of the last two."""
import math
from types import SimpleNamespace

import pytest
import torch

from param_decomp_b200.ops.elementwise import layer_norm
from param_decomp_b200.ops.embedding import embedding
from param_decomp_b200.ops.native import NativeError
from param_decomp_b200.ops.top_logits import eager_top_kl, eager_top_logits, next_token_loss, top_kl, top_kl_rows, top_logits

F16, BF, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.mark.parametrize("x,w,b", [
    (torch.zeros(2, 8, dtype=F16), None, None),  # types the kernels do not have
    (torch.zeros(2, 8, dtype=torch.float64), None, None),
    (torch.zeros(2, 8), torch.ones(8, dtype=F16), None),
    (torch.zeros(2, 8), torch.ones(8, dtype=BF), torch.zeros(8)),  # scale and shift of two types
    (torch.zeros(2, 8), torch.ones(7), None),
    (torch.zeros(2, 8), torch.ones(1, 8), None),
    (torch.zeros(2, 8), None, torch.zeros(9)),
    (torch.zeros(2, 0), None, None),  # no columns, too many, no axis
    (torch.zeros(1, 12289), None, None),
    (torch.zeros(()), None, None),
])
def test_layer_norm_refusals(x, w, b):
    with pytest.raises(ValueError, match="layer_norm"):
        layer_norm(x, w, b, 1e-5)


@pytest.mark.parametrize("tokens,table,out", [
    (torch.zeros(3, dtype=torch.int16), torch.zeros(4, 8), None),
    (torch.zeros(3), torch.zeros(4, 8), None),
    (torch.zeros(3, dtype=torch.int64), torch.zeros(4, 8, dtype=F16), None),
    (torch.zeros(3, dtype=torch.int64), torch.zeros(4, 8, 2), None),
    (torch.zeros(3, dtype=torch.int64), torch.zeros(0, 8), None),
    (torch.zeros(3, dtype=torch.int64), torch.zeros(4, 0), None),
    (torch.zeros(3, dtype=torch.int64), torch.zeros(4, 8), F16),
    (torch.zeros(1, dtype=torch.int64).expand(1 << 30), torch.zeros(4, 8), None),
])
def test_embedding_refusals(tokens, table, out):
    with pytest.raises(ValueError, match="embedding"):
        embedding(tokens, table, 1.0, out)


@pytest.mark.parametrize("logits,k,T", [
    (torch.zeros(2, 8, dtype=F16), 1, 1.0), (torch.zeros(2, 8), 0, 1.0), (torch.zeros(2, 8), 9, 1.0), (torch.zeros(2, 300), 257, 1.0),
    (torch.zeros(2, 8), 1, 0.0), (torch.zeros(2, 8), 1, -1.0), (torch.zeros(2, 8), 1, math.inf), (torch.zeros(2, 8), 1, math.nan),
    (torch.zeros(2, 0), 1, 1.0), (torch.zeros(()), 1, 1.0),
])
def test_top_logits_refusals(logits, k, T):
    with pytest.raises(ValueError, match="top_logits"):
        top_logits(logits, k, T)


_IDX = torch.zeros(2, 3, dtype=torch.int64)


@pytest.mark.parametrize("logits,indices,values,tail,T", [
    (torch.zeros(2, 8, dtype=F16), _IDX, torch.zeros(2, 3), None, 1.0),
    (torch.zeros(2, 8), _IDX.to(torch.int16), torch.zeros(2, 3), None, 1.0),
    (torch.zeros(2, 8), _IDX[:1], torch.zeros(1, 3), None, 1.0),
    (torch.zeros(2, 8), _IDX[:, 0], torch.zeros(2), None, 1.0),
    (torch.zeros(2, 8), _IDX, torch.zeros(2, 2), None, 1.0),
    (torch.zeros(2, 8), _IDX, torch.zeros(2, 3, dtype=F16), None, 1.0),
    (torch.zeros(2, 8), _IDX[:, :0], torch.zeros(2, 0), None, 1.0),
    (torch.zeros(2, 8), torch.zeros(2, 257, dtype=torch.int64), torch.zeros(2, 257), None, 1.0),
    (torch.zeros(2, 8), _IDX, torch.zeros(2, 3), torch.zeros(2, 1), 1.0),
    (torch.zeros(2, 8), _IDX, torch.zeros(2, 3), torch.zeros(2, dtype=BF), 1.0),
    (torch.zeros(2, 8), _IDX, torch.zeros(2, 3), None, 0.0),
])
def test_top_kl_refusals(logits, indices, values, tail, T):
    for call in (top_kl, top_kl_rows):
        with pytest.raises(ValueError, match="top_kl"):
            call(logits, indices, values, tail, T)


def test_tensors_on_the_host_are_refused():
    z, idx = torch.zeros(2, 8), torch.zeros(2, 3, dtype=torch.int64)
    for call in (lambda: layer_norm(z, None, None, 1e-5), lambda: embedding(idx, z), lambda: top_logits(z, 1),
                 lambda: top_kl(z, idx, torch.zeros(2, 3)), lambda: next_token_loss(z, idx[:, 0])):
        with pytest.raises(NativeError, match="cpu"):
            call()


def test_eager_top_logits_breaks_ties_by_column():
    z = torch.tensor([[1.0, 3.0, 3.0, 2.0, 3.0], [0.0, -0.0, -1.0, 0.0, float("-inf")]])
    top = eager_top_logits(z, 2)
    assert top.indices.tolist() == [[1, 2], [0, 1]] and top.values.tolist() == [[3.0, 3.0], [0.0, 0.0]]
    want = torch.tensor([math.log(math.exp(1) + math.exp(2) + math.exp(3)), math.log(1 + math.exp(-1))])
    torch.testing.assert_close(top.tail, want)
    assert eager_top_logits(z, 5).tail.tolist() == [-math.inf, -math.inf]


@pytest.mark.parametrize("k", [1, 4, 19, 20])
def test_eager_top_kl_is_a_divergence_of_events(k):
    g = torch.Generator().manual_seed(k)
    teacher, z = torch.randn(5, 20, generator=g, dtype=torch.float64), torch.randn(5, 20, generator=g, dtype=torch.float64)
    order = torch.sort(teacher, 1, descending=True)[1]
    p, q = (torch.softmax(t, 1).gather(1, order) for t in (teacher, z))
    pe, qe = (torch.cat([t[:, :k], t[:, k:].sum(1, keepdim=True)], 1)[:, :k + (k < 20)] for t in (p, q))
    want = (pe * (pe / qe).log()).sum(1)
    top = eager_top_logits(teacher, k)
    # the tail is kept in fp32: off by 2^-24 of its size
    torch.testing.assert_close(eager_top_kl(z, top.indices, top.values, top.tail), want, atol=1e-6, rtol=0)
    leaf = z.requires_grad_(True)
    assert torch.autograd.gradcheck(lambda t: eager_top_kl(t, top.indices, top.values, top.tail, 2.0), (leaf,))


def test_eager_top_kl_of_one_slot_is_cross_entropy():
    g = torch.Generator().manual_seed(0)
    z, target = torch.randn(6, 11, generator=g, requires_grad=True), torch.tensor([3, 0, -1, 10, -1, 3])
    loss = eager_top_kl(z, target[:, None], torch.zeros(6, 1))
    want = torch.nn.functional.cross_entropy(z, target, ignore_index=-1, reduction="none")
    torch.testing.assert_close(loss, want)
    ours, theirs = (torch.autograd.grad(t.sum(), (z,))[0] for t in (loss, want))
    torch.testing.assert_close(ours, theirs)


def _lm_config(edge: dict, backend: str = "eager_torch", dtype: str = "float32") -> dict:
    import copy

    import __graft_entry__ as ge

    c = copy.deepcopy(ge.SMOKE_CONFIG)
    c["runtime"]["backend"] = backend
    c["target"]["output_edge"] = edge
    c["target"]["weights_dtype"] = dtype
    c["target"]["attention_implementation"] = "xla" if dtype == "float32" else "flash"
    return c


def test_output_edge_of_top_logits_parses_and_is_bounded():
    from pydantic import ValidationError

    from param_decomp_b200.config.experiments import LMExperimentConfig

    cfg = LMExperimentConfig.model_validate(_lm_config({"kind": "top_logits", "k": 16}))
    assert cfg.target.output_edge.k == 16
    for k in (0, 257):
        with pytest.raises(ValidationError):
            LMExperimentConfig.model_validate(_lm_config({"kind": "top_logits", "k": k}))


def test_output_edge_of_top_logits_on_the_eager_backend():
    """The model's loss against the clean side's top logits is `eager_top_kl` of them, chunk by chunk; with all of the
    vocabulary it is the loss of the materialised edge, and so is its gradient."""
    from types import SimpleNamespace

    from param_decomp_b200.config.experiments import TransformerArchConfig
    from param_decomp_b200.models import transformer as tf

    arch = TransformerArchConfig(family="glu_transformer", n_layer=1, d_model=16, n_head=2, d_ff=24, vocab_size=40, max_seq_len=8)
    w = tf.random_init_weights(arch, 0, torch.float32)
    g = torch.Generator().manual_seed(1)
    hc, hm = torch.randn(2, 7, 16, generator=g) * 20, torch.randn(2, 7, 16, generator=g) * 20
    grads, losses = [], []
    for n_top in (None, 40, 5):
        model = tf.TransformerDecomposedModel(arch, w, {}, attention="xla", n_top_logits=n_top, kl_token_chunk=4)
        leaf = hm.clone().requires_grad_(True)
        clean = SimpleNamespace(output=hc, aux={"clean_stats": model._clean_logit_stats(hc)})
        loss = model.recon_loss(clean, SimpleNamespace(output=leaf))
        grads.append(torch.autograd.grad(loss, (leaf,))[0])
        losses.append(loss.detach())
    torch.testing.assert_close(losses[1], losses[0])
    torch.testing.assert_close(grads[1], grads[0], atol=1e-6, rtol=1e-4)
    assert 0 < float(losses[2]) <= float(losses[0])


def test_pretraining_on_native_kernels_needs_a_gpu(tmp_path):
    from param_decomp_b200.pretrain.train import PretrainConfig, pretrain

    cfg = PretrainConfig.model_validate(dict(run_name="t", global_batch=2, num_iterations=1, learning_rate=1e-3, kernels="native",
                                             model=dict(vocab_size=11, n_layer=1, n_head=1, n_embd=8, n_ctx=4)))
    with pytest.raises(ValueError, match="native"):
        pretrain(cfg, tmp_path, run_id="t-00000009")


def test_a_missing_extension_is_said_aloud(monkeypatch, tmp_path):
    from param_decomp_b200.ops import native

    monkeypatch.setattr(native, "AUTOGRAD_PATH", tmp_path / "pd_autograd.so")
    monkeypatch.setattr(native, "_autograd", None)
    with pytest.raises(NativeError, match="ops.build"):
        native.autograd()


@pytest.mark.parametrize("T", [2.0**-121, 2.0**121, 1e-300, 1e300])
def test_temperatures_whose_inverse_leaves_fp32_are_refused(T):
    z = torch.zeros(2, 8)
    for call in (lambda: top_logits(z, 1, T), lambda: top_kl(z, _IDX, torch.zeros(2, 3), None, T),
                 lambda: top_kl_rows(z, _IDX, torch.zeros(2, 3), None, T)):
        with pytest.raises(ValueError, match="temperature"):
            call()


@pytest.mark.parametrize("T", [0.5, 0.7, 1.0, 3.0])
def test_eager_top_kl_of_rows_of_the_lowest_value(T):
    """Teacher or student masked in every place with the type's lowest value: a level row, whatever the temperature makes of it."""
    low = torch.finfo(F32).min
    z, t, idx = torch.zeros(3, 4), torch.zeros(3, 2), torch.tensor([[0, 2]] * 3)
    z[1], t[2] = low, low
    loss = eager_top_kl(z, idx, t, None, T)
    torch.testing.assert_close(loss, torch.full((3,), math.log(2.0)))


def test_evaluated_divergences_do_not_depend_on_the_output_edge():
    """`kl/<variant>` is the divergence over the whole vocabulary; the loss of the edge is its own."""
    from param_decomp_b200.config.experiments import LMExperimentConfig
    from param_decomp_b200.core.objective import build_objective
    from param_decomp_b200.core.run import init_train_state
    from param_decomp_b200.core.train import StepContext
    from param_decomp_b200.evals.lm import ce_and_kl
    from param_decomp_b200.experiments.lm.build import build_lm_run

    results, edge_loss = [], []
    for edge in ({"kind": "materialized"}, {"kind": "top_logits", "k": 3}):
        cfg = LMExperimentConfig.model_validate(_lm_config(edge))
        run = build_lm_run(cfg, None, "cpu")
        obj = build_objective(cfg.pd)
        ctx = StepContext.build(run.model, obj, cfg.pd, lazy_masks=False)
        state = init_train_state(run.model, run.ci_fn, cfg.pd, obj, torch.device("cpu"), cfg.pd.batch_size, cfg.data.seq_len)
        batch = run.sample_eval(0)
        results.append(ce_and_kl(ctx, state, batch))
        clean = run.model.clean_forward(batch)
        half = SimpleNamespace(output=clean.output * 0.5)
        edge_loss.append(float(run.model.recon_loss(clean, half)))
    assert results[0] == results[1] and results[0]["kl/zero_masked"] > 0
    assert 0 < edge_loss[1] < edge_loss[0]


@pytest.mark.parametrize("family", ["moe", "qwen35_moe"])
def test_output_edge_of_top_logits_on_mixture_and_hybrid_targets(family):
    """The edge is wired: a step trains with it, its loss is the divergence from the clean side's top logits, and with k above
    the vocabulary's size that over the whole vocabulary."""
    from param_decomp_b200.config.experiments import LMExperimentConfig
    from param_decomp_b200.core.objective import build_objective
    from param_decomp_b200.core.run import init_train_state
    from param_decomp_b200.core.train import StepContext, train_step
    from param_decomp_b200.experiments.lm.build import build_lm_run
    from param_decomp_b200.models import qwen35
    from tests.test_moe import moe_cfg
    from tests.test_qwen35 import _config

    cs = {k: (12 if k.startswith("experts_") else 8) for k in qwen35.KIND_ORDER}
    raw = (moe_cfg() if family == "moe" else _config(cs)).model_dump(mode="json")
    raw["cadence"] = {"checkpointing": {"kind": "none"}}
    for k in (5, 200):
        raw["target"]["output_edge"] = {"kind": "top_logits", "k": k}
        cfg = LMExperimentConfig.model_validate(raw)
        run = build_lm_run(cfg, None, "cpu")
        assert run.model.n_top_logits == k
        obj = build_objective(cfg.pd)
        ctx = StepContext.build(run.model, obj, cfg.pd, lazy_masks=True)
        state = init_train_state(run.model, run.ci_fn, cfg.pd, obj, torch.device("cpu"), cfg.pd.batch_size, cfg.data.seq_len)
        assert math.isfinite(float(train_step(ctx, state, run.sample_train(0))["loss/total"]))
        with torch.no_grad():
            clean = run.model.clean_forward(run.sample_eval(0))
        masked = SimpleNamespace(output=clean.output * 0.5)
        loss, whole = run.model.recon_loss(clean, masked), run.model.output_kl(clean, masked)
        logits = run.model.logits(clean.output).flatten(0, -2)
        top = eager_top_logits(logits, min(k, logits.shape[-1]))
        assert top.values.shape == clean.aux["clean_stats"]["top"].values.shape
        want = eager_top_kl(run.model.logits(masked.output).flatten(0, -2), top.indices, top.values, top.tail).mean()
        torch.testing.assert_close(loss, want)
        if k == 200:
            torch.testing.assert_close(loss, whole)
        else:
            assert 0 < float(loss) < float(whole)
