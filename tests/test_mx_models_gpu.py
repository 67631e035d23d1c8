"""Models with microscaled layers (``--quantization mxfp4``) on the GPU: every call of an operator that they make against 64 bits, captured
steps against eager ones, and the expert block of gpt-oss through its own layer.  (Log-probabilities are not compared with another
machine's: where 16-bit roundings differ, an activation goes to the neighbouring 8-bit element, 2^-3 of it.)"""
from collections import Counter

import pytest
import torch

from tests import mx_oracle as oracle
from tests.test_mx_gpu import SUM, check_product, check_rows, expert_block, gated_slack
from vllm_distributed_amd import LLM, SamplingParams, ops
from vllm_distributed_amd.parallel import state as pstate

pytestmark = pytest.mark.gpu
PROMPTS = [[5, 9, 200, 17], list(range(10, 90)), [7] * 33]


def generate(tokens, prompts=PROMPTS, **kw):
    kw = dict(dict(dtype="bfloat16", gpu_memory_utilization=0.3), **kw)
    llm = LLM(max_model_len=256, block_size=16, num_gpu_blocks_override=64, max_num_seqs=8, quantization="mxfp4", load_format="dummy", **kw)
    try:
        runner = llm.engine.core.executor.driver.worker.model_runner
        layer = next(iter(runner.model.layers.values()))
        assert getattr(layer.mlp, "mx13_qw", None) is not None or layer.mlp.down_proj.takes_rows8
        out = llm.generate(prompts, SamplingParams(temperature=0.0, max_tokens=tokens, ignore_eos=True, logprobs=20))
        return [(o.outputs[0].token_ids, o.outputs[0].logprobs) for o in out], bool(runner.graphs)
    finally:
        llm.shutdown()
        pstate.destroy_model_parallel()


def dense(w):
    """The weight's numbers in 64 bits on the CPU."""
    from vllm_distributed_amd.ops import quant
    return quant.mx_weight_dense(ops.MxWeight(w.qw.cpu(), w.ws.cpu(), w.rows)).double()


def numbers(x):
    return ops.mx_dequantize(x, torch.float32).cpu().double() if isinstance(x, ops.MxRows) else oracle.blocks(x, 8)[2]


def watch(monkeypatch, seen):
    """Every microscaled call that a model makes, against 64 bits over the operands it got, with the bounds of the operators' own tests."""
    real = {n: getattr(ops, n) for n in ("mx_linear", "mx_linear_partials", "mx_gate_up", "mx_experts", "mx_experts_routed", "rms_norm_mx",
                                         "fused_add_rms_norm_mx", "reduce_add_rms_norm_mx")}

    def product(x, w, bias=None):
        y = real["mx_linear"](x, w, bias)
        if y.shape[0] <= 128:
            check_product(y, numbers(x), dense(w)[:, :x.shape[1]], y.dtype, None if bias is None else bias.cpu())
            seen["mx_linear"] += 1
        return y

    def partials(x, w):
        slabs = real["mx_linear_partials"](x, w)
        if slabs is not None and x.shape[0] <= 128:
            xv, wv = numbers(x), dense(w)[:, :x.shape[1]]
            assert ((slabs.double().sum(0).cpu() - xv @ wv.T).abs() <= SUM * (xv.abs() @ wv.abs().T)).all()
            seen["mx_linear_partials"] += 1
        return slabs

    def gate_up(x, w, *args):
        r = real["mx_gate_up"](x, w, *args)
        if r.shape[0] <= 128:
            check_rows(r, *gated_slack(numbers(x), dense(w)[:, :x.shape[1]], None, 0.0))
            seen["mx_gate_up"] += 1
        return r

    def norm(name, slabs=False):
        def call(x, *args):
            out = real[name](x, *args)
            residual = args[0] if len(args) == 3 else None
            r = out if residual is None else out[0]
            if r.shape[0] <= 128:
                parts = (x.double().cpu() if slabs else x.double().cpu().unsqueeze(0))
                if residual is not None:
                    parts = torch.cat([parts, residual.double().cpu().unsqueeze(0)])
                total = parts.sum(0)
                v = total / torch.sqrt((total ** 2).mean(-1, keepdim=True) + args[-1]) * args[-2].double().cpu()
                size = parts.abs().sum(0) / total.abs().clamp_min(1e-30) if slabs else torch.ones_like(v)
                check_rows(r, v, (40 + (len(parts) + 1) * size) * 2.0 ** -24 * v.abs())
                seen[name] += 1
            return out
        return call

    def experts(x, topw, topi, w13, w2, b13=None, b2=None, bias13=None, bias2=None, limit=0.0, **kw):
        y = real["mx_experts"](x, topw, topi, w13, w2, bias13, bias2, limit=limit, **kw)
        if x.shape[0] <= 128:
            v13, v2, inter = dense(w13)[..., :x.shape[1]], dense(w2), w13.rows // 2
            want, bound = expert_block(numbers(x), topw.cpu(), topi.cpu(), v13, v2[..., :inter], bias13, bias2, limit)
            off = (y.cpu().double() - want).abs()
            assert (off <= bound).all(), f"worst {(off / bound).max():.3g} of the bound"
            seen["mx_experts"] += 1
        return y

    def routed(logits, x, k, renormalize, w13, w2, bias13=None, bias2=None, limit=0.0, **kw):
        y = real["mx_experts_routed"](logits, x, k, renormalize, w13, w2, bias13=bias13, bias2=bias2, limit=limit, **kw)
        if x.shape[0] <= 16:
            topw, topi = ops.moe_topk(logits.sum(0) if logits.dim() == 3 else logits, k, renormalize)
            want, bound = expert_block(numbers(x), topw.cpu(), topi.cpu(), dense(w13)[..., :x.shape[1]], dense(w2)[..., :w13.rows // 2], bias13,
                                       bias2, limit)
            # (sums of the router's parts in another order: the weights are off by a few 2^-24 times the logits' size)
            off = (y.cpu().double() - want).abs()
            assert (off <= bound + 2.0 ** -18 * want.abs()).all(), f"worst {(off / bound).max():.3g} of the bound"
            seen["mx_experts_routed"] += 1
        return y
    for name, f in (("mx_linear", product), ("mx_linear_partials", partials), ("mx_gate_up", gate_up), ("mx_experts", experts), ("mx_experts_routed", routed),
                    ("rms_norm_mx", norm("rms_norm_mx")), ("fused_add_rms_norm_mx", norm("fused_add_rms_norm_mx")),
                    ("reduce_add_rms_norm_mx", norm("reduce_add_rms_norm_mx", True))):
        monkeypatch.setattr(ops, name, f)


LINEARS = {"mx_linear", "rms_norm_mx", "fused_add_rms_norm_mx"}
WIDE = dict(num_hidden_layers=2, num_key_value_heads=2, head_dim=64)


@pytest.mark.parametrize("model,over,calls", [
    ("llama-tiny", {}, LINEARS | {"mx_gate_up"}),
    # reductions long enough to be split over the grid: the sums go to the norm behind the projection, or to the rotation behind q, k and v
    ("llama-tiny", dict(WIDE, hidden_size=512, num_attention_heads=64, intermediate_size=4096), LINEARS | {"mx_gate_up", "mx_linear_partials", "reduce_add_rms_norm_mx"}),
    ("llama-tiny", dict(WIDE, hidden_size=4096, num_attention_heads=4, intermediate_size=4096), LINEARS | {"mx_gate_up", "mx_linear_partials"}),
    ("mixtral-tiny", {}, LINEARS | {"mx_experts", "mx_experts_routed"}), ("qwen3-moe-tiny", {}, LINEARS | {"mx_experts", "mx_experts_routed"}),
    ("gpt-oss-tiny", {}, {"mx_experts", "mx_experts_routed"}),
    ("glm4-moe-tiny", {}, LINEARS | {"mx_experts"}), ("phimoe-tiny", {}, {"mx_linear", "mx_experts"}), ("stablelm-tiny", {}, {"mx_linear", "mx_gate_up"})])
def test_every_call_of_a_model(model, over, calls, monkeypatch):
    seen = Counter()
    watch(monkeypatch, seen)
    generate(2, model=model, enforce_eager=True, hf_overrides=over)
    assert set(seen) >= calls, seen


@pytest.mark.parametrize("model", ["llama-tiny", "mixtral-tiny", "gpt-oss-tiny"])
def test_captured_steps_are_the_eager_ones(model):
    a, graphs = generate(6, model=model)
    b, _ = generate(6, model=model, enforce_eager=True)
    assert graphs and a == b


@pytest.mark.parametrize("tokens", [1, 7, 64, 300, 1500])
def test_gpt_oss_block(tokens):
    """The block with its biases and the clamp, from matrices as a checkpoint has them (gate and up interleaved), at sizes of each kind of
    tile, against 64 bits behind the router's choice."""
    from vllm_distributed_amd.models.gpt_oss import GptOssMoE
    from vllm_distributed_amd.models.layers.linear import QuantSpec, quantized_linears
    cfg = dict(hidden_size=288, intermediate_size=160, num_local_experts=8, num_experts_per_tok=2, swiglu_limit=7.0)
    gen = torch.Generator().manual_seed(tokens)
    with torch.device("cuda"), quantized_linears(QuantSpec("mxfp4", 32, 1)):
        moe = GptOssMoE(cfg, torch.bfloat16, False)
    moe.gate.weight.data.copy_(torch.randn(8, 288, generator=gen) * 0.1)
    moe.gate.bias.data.zero_()
    m = {kind: (torch.randn(*shape, generator=gen) * 0.06).to(torch.bfloat16) for kind, shape in (
        ("gate_up_proj", (8, 288, 320)), ("gate_up_proj_bias", (8, 320)), ("down_proj", (8, 160, 288)), ("down_proj_bias", (8, 288)))}
    for kind, w in m.items():
        moe.load_stacked(kind, w)
    moe.finalize_weights()
    x = torch.randn(tokens, 288, generator=gen).to(torch.bfloat16)
    y = moe(x.cuda())
    topw, topi = ops.moe_topk(moe.gate(x.cuda()), 2, True)
    apart = lambda w: torch.cat([w[..., 0::2], w[..., 1::2]], -1)
    v13 = torch.stack([oracle.blocks(w.t(), 4)[2] for w in apart(m["gate_up_proj"])])
    v2 = torch.stack([oracle.blocks(w.t(), 4)[2] for w in m["down_proj"]])
    want, bound = expert_block(oracle.blocks(x, 8)[2], topw.cpu(), topi.cpu(), v13, v2, apart(m["gate_up_proj_bias"]), m["down_proj_bias"], 7.0)
    off = (y.cpu().double() - want).abs()
    assert (off <= bound).all(), f"worst {(off / bound).max():.3g} of the bound"
