"""Microscaled rows, weights and layers on the CPU: the definition against 64 bits, the layout, refusals, and models whose layers are
microscaled (``--quantization mxfp4``)."""
import json
from types import SimpleNamespace

import pytest
import torch

from tests import mx_oracle as oracle
from vllm_distributed_amd import LLM, SamplingParams, ops
from vllm_distributed_amd.config import ModelConfig
from vllm_distributed_amd.ops import quant
from vllm_distributed_amd.parallel import state as pstate


def rows(m, k, seed=0, dtype=torch.float32):
    gen = torch.Generator().manual_seed(seed + m * 7 + k)
    return (torch.randn(m, k, generator=gen) * torch.exp(2 * torch.randn(m, k, generator=gen))).to(dtype)


# ------------------------------------------------------------------ the format
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k", [(0, 64), (1, 32), (5, 96), (33, 544)])
def test_quantize_and_back(bits, dtype, m, k):
    x = rows(m, k, dtype=dtype)
    if m > 2:
        x[1] = 0
        x[2, 3], x[2, 40] = float("nan"), float("-inf")
    r = ops.mx_quantize(x, bits)
    code, byte, value = oracle.blocks(x, bits)
    assert r.shape == (m, k) and r.dtype == dtype and torch.equal(r.s.view(torch.uint8).long(), byte)
    back = ops.mx_dequantize(r, torch.float32)
    assert torch.equal(back.nan_to_num(7777.0), value.float().nan_to_num(7777.0))
    if bits == 4:
        keep = (byte != 255).repeat_interleave(32, 1)
        got = torch.stack([r.q & 15, r.q >> 4], -1).reshape(m, k).long()
        assert torch.equal(got[keep], code[keep])


def test_the_scale_is_the_smallest_that_holds_a_block():
    x = torch.zeros(6, 32)
    x[:, 0] = torch.tensor([6.0, 6.0001, 3.0, 448.0, 449.0, 2.0 ** -140])
    assert ops.mx_quantize(x, 4).s.view(torch.uint8).flatten().tolist() == [127, 128, 126, 134, 134, 0]
    assert ops.mx_quantize(x, 8).s.view(torch.uint8).flatten().tolist() == [121, 121, 120, 127, 128, 0]


@pytest.mark.parametrize("lead", [(), (3,)])
@pytest.mark.parametrize("halves,n", [(1, 8), (1, 24), (1, 160), (2, 16), (2, 96), (2, 512)])
@pytest.mark.parametrize("k", [32, 160, 544])
def test_pack_and_unpack(lead, halves, n, k):
    gen = torch.Generator().manual_seed(n + k)
    q = torch.randint(0, 256, (*lead, n, k // 2), generator=gen, dtype=torch.uint8)
    s = torch.randint(0, 255, (*lead, n, k // 32), generator=gen, dtype=torch.uint8)
    w = quant.pack_mx(q, s, halves=halves)
    assert w.rows == (n if halves == 1 else 2 * ((n // 2 + 127) // 128 * 128))
    uq, us = quant.unpack_mx(w)
    half, step = n // halves, w.rows // halves
    for i in range(halves):
        assert torch.equal(uq[..., i * step:i * step + half, :k // 2], q[..., i * half:(i + 1) * half, :])
        assert torch.equal(us[..., i * step:i * step + half, :k // 32], s[..., i * half:(i + 1) * half, :])
        assert not uq[..., i * step + half:(i + 1) * step, :].any()
    assert not uq[..., k // 2:].any()
    b = torch.randn(*lead, n)
    p = quant.pad_mx_bias(b, halves)
    if halves == 2:
        assert p.shape[-1] == w.rows and torch.equal(p[..., :half], b[..., :half]) and torch.equal(p[..., step:step + half], b[..., half:])


# ------------------------------------------------------------------ products (32-bit sums of exact products: k roundings of 2^-24)
@pytest.mark.parametrize("m,n,k", [(1, 8, 32), (3, 40, 96), (7, 136, 544)])
def test_products(m, n, k):
    x = rows(m, k)
    gen = torch.Generator().manual_seed(5)
    q, s, wv = oracle.random_weight(n, k, gen)
    b = torch.randn(n)
    xv = oracle.blocks(x, 8)[2]
    y = ops.mx_linear(x, quant.pack_mx(q, s), b)
    assert ((y.double() - (xv @ wv.T + b.double())).abs() <= (k + 2) * 2.0 ** -24 * (xv.abs() @ wv.abs().T + b.abs().double())).all()
    assert torch.equal(ops.mx_linear(x.view(1, m, k), quant.pack_mx(q, s), b)[0], y)


@pytest.mark.parametrize("limit", [0.0, 7.0])
def test_experts_are_their_products(limit):
    """The sparse block against the layer's own product and gate, expert by expert; a slot of another rank's expert adds nothing."""
    t, e, k, h, inter = 9, 4, 2, 64, 96
    gen = torch.Generator().manual_seed(1)
    x = rows(t, h) * 0.1
    ws13 = [oracle.random_weight(2 * inter, h, gen, 1) for _ in range(e)]
    ws2 = [oracle.random_weight(h, inter, gen, 1) for _ in range(e)]
    pack = lambda ws, halves: quant.pack_mx(torch.stack([w[0] for w in ws]), torch.stack([w[1] for w in ws]), halves=halves)
    b13, b2 = torch.randn(e, 2 * inter), torch.randn(e, h)
    topi = torch.stack([torch.randperm(e, generator=gen)[:k] for _ in range(t)]).int()
    topw = torch.rand(t, k)
    w13, w2, pb = pack(ws13, 2), pack(ws2, 1), quant.pad_mx_bias(b13, 2)
    y = ops.mx_experts(x, topw, topi, w13, w2, pb, b2, limit=limit)
    want = torch.zeros(t, h)
    for i in range(t):
        for j in range(k):
            c = int(topi[i, j])
            a = ops.mx_gate_up(x[i:i + 1], ops.MxWeight(w13.qw[c], w13.ws[c], w13.rows), pb[c], limit=limit)
            want[i] += topw[i, j] * ops.mx_linear(a, ops.MxWeight(w2.qw[c], w2.ws[c], h), b2[c])[0]
    assert torch.allclose(y, want, rtol=1e-5, atol=1e-5)
    part = lambda w, sl: ops.MxWeight(w.qw[sl].contiguous(), w.ws[sl].contiguous(), w.rows)
    halves = [ops.mx_experts(x, topw, topi, part(w13, sl), part(w2, sl), pb[sl], b2[sl], expert_start=sl.start, local_experts=2,
                             num_experts=e, limit=limit) for sl in (slice(0, 2), slice(2, 4))]
    assert torch.allclose(halves[0] + halves[1], y, rtol=1e-5, atol=1e-5)


def test_refusals():
    x = rows(4, 128)
    q, s, _ = oracle.random_weight(64, 128, torch.Generator().manual_seed(0))
    w = quant.pack_mx(q, s)
    r = ops.mx_quantize(x)
    e3 = ops.MxWeight(w.qw.unsqueeze(0), w.ws.unsqueeze(0), 64)
    gen = torch.Generator().manual_seed(1)
    g1 = quant.pack_mx(*[t.unsqueeze(0) for t in oracle.random_weight(256, 128, gen)[:2]], halves=2)
    k2 = quant.pack_mx(*[t.unsqueeze(0) for t in oracle.random_weight(64, 256, gen)[:2]])
    topw, topi = torch.ones(4, 1), torch.zeros(4, 1, dtype=torch.int32)
    assert ops.mx_experts(x, topw, topi, g1, e3).shape == (4, 64)
    for call, error in (
            (lambda: ops.mx_quantize(x, 5), ValueError), (lambda: ops.mx_quantize(x[:, :40]), ValueError),
            (lambda: ops.mx_quantize(x[:, :0]), ValueError), (lambda: ops.mx_quantize(x.double()), TypeError),
            (lambda: ops.mx_quantize(x.long()), TypeError), (lambda: ops.mx_dequantize(r, torch.float64), TypeError),
            (lambda: ops.rms_norm_mx(x[:, :48], torch.ones(48), 1e-5), ValueError),
            (lambda: ops.mx_linear(x[:, :96].contiguous().repeat(1, 3), w), ValueError),
            (lambda: ops.mx_linear(ops.mx_quantize(x, 4), w), ValueError), (lambda: ops.mx_linear(x[:, :40], w), ValueError),
            (lambda: ops.mx_gate_up(x, w), ValueError),
            (lambda: ops.mx_experts(x, topw, topi, g1, e3, local_experts=1), ValueError),
            (lambda: ops.mx_experts(x, topw, topi, g1, e3, local_experts=2, num_experts=4), ValueError),
            (lambda: ops.mx_experts(x, topw, topi, g1, e3, num_experts=2), ValueError),
            (lambda: ops.mx_experts(x, topw, topi, g1, e3, expert_start=1), ValueError),
            (lambda: ops.mx_experts(x, topw, topi, g1, e3, expert_start=4, local_experts=1, num_experts=4), ValueError),
            (lambda: ops.mx_experts(x, topw, topi, g1, k2), ValueError), (lambda: ops.mx_experts(x, topw, topi, e3, e3), ValueError),
            (lambda: ops.mx_experts(x[:3], topw, topi, g1, e3), ValueError),
            (lambda: ops.mx_experts(x, topw, topi[:, :0], g1, e3), ValueError),
            (lambda: quant.pack_mx(q[:60], s[:60]), ValueError), (lambda: quant.pack_mx(q[:24], s[:24], halves=2), ValueError),
            (lambda: quant.pack_mx(q, s[:, :3]), ValueError), (lambda: quant.pack_mx(q.int(), s), ValueError),
            (lambda: ops.MxRows.of(r.q, r.s[:3], torch.float32), ValueError),
            (lambda: ops.MxRows.of(r.q.view(torch.int8), r.s, torch.float32), TypeError)):
        with pytest.raises(error):
            call()


def one_row_views(dtype):
    """[1, 64] views whose row stride torch leaves as it was: rows of a matrix 523 wide from the front, the middle and an odd address, a column
    turned, an expanded row, a part of a longer row, and leading dimensions."""
    base = rows(5, 523, dtype=dtype)
    column = rows(64, 1, dtype=dtype)
    return [base[:1, :64], base[1:2, 5:69], base[4:, 8:72], column.t(), column.flatten().expand(1, 64), base[:1].as_strided((1, 64), (0, 1)),
            base[2:3, :128:2], base[3:4, None, :64]]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_one_row_of_any_stride_is_a_row(dtype):
    """What the kernels get: rows at 16-byte borders, their stride a multiple of eight that holds them, however many there are."""
    from vllm_distributed_amd.ops import hip
    views = one_row_views(dtype)
    assert len({v.stride() for v in views}) > 3
    base = rows(6, 523, dtype=dtype)
    for x in views + [base[:, :64], base[::2, 3:67], base[:1, :64].expand(3, 64), base[:0, :64]]:
        got = hip._mx_rows(x)
        assert torch.equal(got, x.reshape(-1, 64))
        if got.shape[0]:
            assert got.stride(1) == 1 and got.stride(0) % 8 == 0 and got.stride(0) >= 64 and got.data_ptr() % 16 == 0, (x.stride(), got.stride())
    keep = base.new_zeros(3, 72)[:1, :64]                        # (nothing is copied that can be read as it is)
    assert hip._mx_rows(keep).data_ptr() == keep.data_ptr()


def test_norm_kernel_gets_operands_at_16_byte_borders(monkeypatch):
    """A branch or a residual from an odd address is copied; one that can be read as it is is not."""
    from vllm_distributed_amd.ops import hip
    seen = []
    monkeypatch.setattr(hip, "_LIB", SimpleNamespace(vdamd_mx_rms_norm=lambda *a: seen.append(a) or 0))
    monkeypatch.setattr(hip, "_mx_device", lambda *a: None)
    monkeypatch.setattr(hip, "_stream", lambda: 0)
    m, h = 3, 64
    gain = torch.ones(h, dtype=torch.bfloat16)
    flat = rows(1, (m + 1) * h, dtype=torch.bfloat16).flatten()
    for at in (0, 1, 4, 8):
        x, residual = flat[8:8 + m * h].view(m, h), flat[at:at + m * h].view(m, h)
        _, out = hip.mx_rms_norm(x, None, residual, gain, 1e-5)
        # (the C entry's order: q, ldq, s, lds, residual_out, x, ldx, slabs, ks, residual, ..)
        q, residual_out, x_at, residual_at = (seen[-1][i] for i in (0, 4, 5, 9))
        assert not (q | residual_out | x_at | residual_at) % 16
        assert (residual_at == residual.data_ptr()) == (at % 8 == 0) and out.shape == residual.shape


@pytest.mark.parametrize("m", [1, 256, 2000, 4096, 8131, 12288, 20000])
def test_large_tiles_are_expected_to_take_the_rounds_that_they_take(m):
    """The plan's expected time of 256-row tiles against the launch, dealt out as the kernel does: eight dies, each with its own tile columns
    and at most 32 workgroups, one tile after the other."""
    from vllm_distributed_amd.ops import hip
    for n in (8, 264, 512, 1000, 1280, 2880, 4104, 5120, 6144, 10240, 57344):
        for kb in (1, 9, 64):
            ntm, ntn = (m + 255) // 256, (n + 255) // 256
            per_die = min(ntm * ((ntn + 7) // 8), 32)
            tiles = [ntm * ((ntn * (d + 1) >> 3) - (ntn * d >> 3)) for d in range(8)]
            rounds = max(len(range(i, t, per_die)) for t in tiles for i in range(per_die))
            got = hip._mx_estimate(m, n, kb, hip.MX_BIG, 0, 1)
            # (a step 1 us, 1.22 on a full chip, 1.4 where a die has one column; 5.4 beside the steps of a tile)
            most = 1.4 if ntn <= 8 else 1.22
            assert rounds * (kb + 5.4) - 1e-6 <= got <= rounds * (most * kb + 5.4) + 1e-6, (n, kb, rounds, got)


def test_narrow_outputs_of_many_rows_go_through_the_ring():
    """Fewer than eight tile columns leave dies without work: us of large tiles and of the ring beside each size."""
    from vllm_distributed_amd.ops import hip
    for m, n, k, gated in ((12288, 1280, 8192, False),      # 184, 129
                           (20000, 264, 4640, False),       # 150, 63
                           (16384, 1000, 1056, False),      # 48, 38
                           (12288, 768, 4096, False),       # 92, 62
                           (16384, 1280, 8192, False),      # 195, 183
                           (6000, 5120, 6144, True)):       # 200, 189
        assert hip.mx_plan(m, n, (k + 127) // 128, True, gated)[0] != hip.MX_BIG, (m, n, k)
    for m, n, k, gated in ((4096, 8192, 28672, False), (4096, 2880, 4096, False), (8192, 6144, 4096, False), (8192, 2048, 8192, False), (6007, 28672, 4096, True)):
        assert hip.mx_plan(m, n, (k + 127) // 128, True, gated) == (hip.MX_BIG, 1), (m, n, k)


# ------------------------------------------------------------------ layers and models
def q8(x):
    return oracle.blocks(x.reshape(-1, x.shape[-1]), 8)[2].view(x.shape)


def q4(w):
    return oracle.blocks(w, 4)[2]


PROMPTS = [[5, 9, 200, 17], list(range(10, 50))]


def generate(tokens=5, check=None, **kw):
    kw = dict(dict(device="cpu", dtype="float32", max_model_len=128, block_size=16, num_gpu_blocks_override=64, max_num_seqs=8), **kw)
    llm = LLM(**kw)
    try:
        if check is not None:
            check(llm.engine.core.executor.driver.worker.model_runner.model)
        out = llm.generate(PROMPTS, SamplingParams(temperature=0.0, max_tokens=tokens, ignore_eos=True, logprobs=20))
    finally:
        llm.shutdown()
        pstate.destroy_model_parallel()
    return [(o.outputs[0].token_ids, o.outputs[0].logprobs) for o in out]


def compare(a, b, tol):
    """Log-probabilities of the first token and, as long as both chose the same ones, of the next."""
    for (ta, la), (tb, lb) in zip(a, b):
        for i in range(len(ta)):
            common = set(la[i]) & set(lb[i])
            assert len(common) >= 15
            assert max(abs(la[i][t] - lb[i][t]) for t in common) <= tol, (i, max(abs(la[i][t] - lb[i][t]) for t in common))
            if ta[i] != tb[i]:
                break


def packed(model):
    for layer in model.layers.values():
        a = layer.self_attn
        assert a.qkv_proj.takes_rows8 and a.o_proj.takes_rows8 and not hasattr(a.qkv_proj, "weight")
        if hasattr(layer.mlp, "mx13_qw"):
            assert layer.mlp.mx13_qw is not None and not hasattr(layer.mlp, "w13")
        else:
            assert layer.mlp.gate_up_proj.takes_rows8 and layer.mlp.down_proj.takes_rows8


@pytest.mark.parametrize("model", ["llama-tiny", "mixtral-tiny", "qwen3-moe-tiny", "gemma-tiny"])
def test_models_are_their_dense_twin_of_quantised_operands(model, monkeypatch):
    """Every linear layer and expert as the product of quantised operands in 64 bits, in the unquantised model.  The two differ where
    32-bit roundings put a value on the other side of the middle of two 8-bit elements: of some 10^6 elements, each with about 2^-24 *
    2^4 of such a chance, a few, by 2^-3 of one among hundreds of summands - 10^-2 of the projections' outputs at most, and log-probabilities
    of small random models move by less than that."""
    from vllm_distributed_amd.models.layers import linear, moe
    got = generate(model=model, quantization="mxfp4", check=packed)
    dense = linear._LinearBase._base_matmul
    experts = moe.FusedMoE._expert_mlp

    def product(x, w, b=None):
        y = q8(x) @ q4(w).T
        return (y if b is None else y + b.double()).float()

    def base(self, x, bias, out=None):
        if type(self) is linear.ReplicatedLinear:
            return dense(self, x, bias, out)
        return product(x, self.weight, bias)

    def expert(self, e, x):
        h = product(x, self.w13[e])
        return product(ops.silu_and_mul(h), self.w2[e])
    monkeypatch.setattr(linear._LinearBase, "_base_matmul", base)
    monkeypatch.setattr(moe.FusedMoE, "_expert_mlp", expert)
    for cls in (linear.ColumnParallelLinear, linear.QKVParallelLinear):
        monkeypatch.setattr(cls, "forward", lambda self, x: self._matmul(x, self.bias))
    monkeypatch.setattr(linear.ColumnParallelLinear, "forward_silu", lambda self, x, rows8=False: None)
    monkeypatch.setattr(linear.RowParallelLinear, "forward_gated", lambda self, g, *a: self.forward(ops.silu_and_mul(g), *a))
    monkeypatch.setattr(linear.RowParallelLinear, "forward_add", lambda *a: False)
    compare(got, generate(model=model), 1e-2)


def test_checkpoint_file_and_dummy_stream_agree(tmp_path):
    from vllm_distributed_amd.models.loader import save_dummy_checkpoint
    save_dummy_checkpoint(ModelConfig(model="mixtral-tiny", dtype="float32", load_format="dummy"), str(tmp_path / "m"))
    a = generate(model="mixtral-tiny", quantization="mxfp4")
    b = generate(model=str(tmp_path / "m"), quantization="mxfp4")
    assert [t for t, _ in a] == [t for t, _ in b]


def test_layers_that_do_not_divide_into_blocks_stay_dense():
    from vllm_distributed_amd.models.layers.linear import QuantSpec, ReplicatedLinear, quantized_linears
    for k, n, mx in ((96, 64, True), (80, 64, False), (96, 60, False)):
        with quantized_linears(QuantSpec("mxfp4", 32, 1)):
            lin = ReplicatedLinear(k, n, True, torch.float32)
        lin.weight.data.normal_()
        lin.bias.data.normal_()
        w = lin.weight.data.clone()
        lin.finalize_weights()
        lin.finalize_weights()                           # (a second call changes nothing)
        assert (lin.mx_qw is not None) == mx and lin.takes_rows8 == mx
        x = rows(3, k)
        want = (q8(x) @ q4(w).T).float() if mx else x @ w.T
        assert torch.allclose(lin(x), want + lin.bias, rtol=1e-4, atol=1e-4 * float(want.abs().max()))


def test_an_adapter_sees_the_sixteen_bit_rows():
    """A projection with an adapter takes its input unquantised: the adapter multiplies it too."""
    from vllm_distributed_amd.models.layers.linear import ColumnParallelLinear, QuantSpec, RowParallelLinear, quantized_linears
    from vllm_distributed_amd.models.llama import LlamaMLP
    with quantized_linears(QuantSpec("mxfp4", 32, 1)):
        mlp = LlamaMLP(64, 128, torch.float32)
    for lin in (mlp.gate_up_proj, mlp.down_proj):
        lin.weight.data.normal_(0, 0.1)
        lin.finalize_weights()
    x = rows(3, 64)
    plain = mlp(x)
    assert isinstance(mlp.gate_up_proj.forward_silu(x, True), ops.MxRows)
    seen = []

    class Slots:
        def apply(self, x, y):
            seen.append(type(x))
            return y
    mlp.down_proj.lora = mlp.gate_up_proj.lora = Slots()
    assert not mlp.down_proj.takes_rows8 and mlp.gate_up_proj.forward_silu(x, mlp.down_proj.takes_rows8) is None
    assert torch.allclose(mlp(x), plain, rtol=1e-4, atol=1e-4) and seen == [torch.Tensor, torch.Tensor]


def gpt_oss_files(tmp_path):
    """The same model twice: experts as blocks, and as the numbers that the blocks stand for."""
    from safetensors.torch import load_file, save_file
    from vllm_distributed_amd.models.gpt_oss import mxfp4_dequantize, mxfp4_quantize
    from vllm_distributed_amd.models.loader import save_dummy_checkpoint
    mc = ModelConfig(model="gpt-oss-tiny", dtype="float32", load_format="dummy")
    wide, blocks = tmp_path / "wide", tmp_path / "blocks"
    save_dummy_checkpoint(mc, str(wide))
    a, b = {}, {}
    for name, t in load_file(str(wide / "model.safetensors")).items():
        if name.endswith((".experts.gate_up_proj", ".experts.down_proj")):
            q, s = mxfp4_quantize(t.transpose(1, 2).contiguous())
            b[name + "_blocks"], b[name + "_scales"] = q, s
            a[name] = mxfp4_dequantize(q, s, torch.float32).transpose(1, 2).contiguous()
        else:
            a[name] = b[name] = t
    save_file(a, str(wide / "model.safetensors"))
    blocks.mkdir()
    save_file(b, str(blocks / "model.safetensors"))
    (blocks / "config.json").write_text(json.dumps(dict(mc.hf_config, quantization_config={"quant_method": "mxfp4"})))
    return str(wide), str(blocks), b


def test_gpt_oss_experts_stay_blocks(tmp_path, monkeypatch):
    """With mxfp4 the blocks of a checkpoint, and blocks made of the numbers they stand for (which are exact), are one model: the
    widened model with quantised rows (the tolerance of the dense twins above).  Without the option nothing is packed."""
    from vllm_distributed_amd.models.gpt_oss import GptOssMoE
    wide, blocks, _ = gpt_oss_files(tmp_path)

    def check(model):
        for layer in model.layers.values():
            assert layer.mlp.mx13_qw is not None and not hasattr(layer.mlp, "w13")
            assert layer.self_attn.qkv_proj.mx_qw is None and not layer.self_attn.qkv_proj.takes_rows8
    a, b = (generate(model=d, quantization="mxfp4", check=check) for d in (blocks, wide))
    assert a == b

    def unpacked(model):
        assert all(layer.mlp.mx13_qw is None for layer in model.layers.values())

    def expert(self, e, x):
        h = (q8(x) @ self.w13[e][:, :self.hidden].double().T).float() + self.b13[e]
        a = self._act(h)[:, :self.inter_local]
        return (q8(a) @ self.w2[e][:, :self.inter_local].double().T).float() + self.b2[e]
    monkeypatch.setattr(GptOssMoE, "_expert_mlp", expert)
    compare(a, generate(model=blocks, check=unpacked), 1e-2)


def test_a_checkpoint_with_a_matrix_missing_is_refused(tmp_path):
    from safetensors.torch import load_file, save_file
    from vllm_distributed_amd.models.loader import save_dummy_checkpoint
    _, blocks, tensors = gpt_oss_files(tmp_path)
    name = next(n for n in tensors if n.endswith("down_proj_blocks"))
    less = {n: t for n, t in tensors.items() if not n.startswith(name[:-len("_blocks")]) or n.endswith("bias")}
    save_file(less, blocks + "/model.safetensors")
    with pytest.raises(Exception, match="not found"):
        generate(model=blocks, quantization="mxfp4")
    pstate.destroy_model_parallel()
    d = str(tmp_path / "llama")
    save_dummy_checkpoint(ModelConfig(model="llama-tiny", dtype="float32", load_format="dummy"), d)
    full = load_file(d + "/model.safetensors")
    save_file({n: t for n, t in full.items() if "layers.1.self_attn.k_proj" not in n}, d + "/model.safetensors")
    with pytest.raises(Exception, match="partly filled"):
        generate(model=d, quantization="mxfp4")
    pstate.destroy_model_parallel()


@pytest.mark.parametrize("model", ["deepseek-v3-tiny", "falcon-tiny", "opt-tiny"])
def test_families_without_such_layers_refuse(model):
    with pytest.raises((NotImplementedError, ValueError), match="mxfp4"):
        generate(model=model, quantization="mxfp4")
    pstate.destroy_model_parallel()


@pytest.mark.slow
@pytest.mark.parametrize("model,saves", [("llama-tiny", True), ("gpt-oss-tiny", False), ("mixtral-tiny", True)])
def test_two_ranks_and_their_saved_shards(model, saves, tmp_path, monkeypatch):
    """Two ranks hold blocks of their rows and columns - the blocks of the whole matrices, since shards end on blocks - and answer as one
    process does; what they save is read back as it is (shards of gpt-oss cannot be saved: two of its names share a tensor)."""
    from vllm_distributed_amd.engine.arg_utils import EngineArgs
    from vllm_distributed_amd.engine.llm_engine import LLMEngine
    from vllm_distributed_amd.models.loader import save_dummy_checkpoint
    from vllm_distributed_amd.utils import get_open_port
    ckpt, shards = str(tmp_path / "ckpt"), str(tmp_path / "shards")
    save_dummy_checkpoint(ModelConfig(model=model, dtype="float32", load_format="dummy"), ckpt)
    for k, v in dict(VLLM_RPC_SECRET="s", VLLM_HOST_IP="127.0.0.1", GLOO_SOCKET_IFNAME="lo",
                     VLLM_HEAD_LOCAL_DEVICES="2", OMP_NUM_THREADS="2").items():
        monkeypatch.setenv(k, v)

    def run(where, load_format, tp=2):
        pstate.destroy_model_parallel()
        monkeypatch.setenv("VLLM_SERVER_PORT", str(get_open_port()))
        eng = LLMEngine.from_engine_args(EngineArgs(
            model=where, device="cpu", dtype="float32", max_model_len=128, block_size=16, load_format=load_format, quantization="mxfp4",
            num_gpu_blocks_override=64, max_num_seqs=8, tensor_parallel_size=tp,
            distributed_executor_backend="distributed" if tp > 1 else "uni"))
        try:
            sp = SamplingParams(temperature=0.0, max_tokens=4, ignore_eos=True, logprobs=20)
            ids = [eng.add_request(None, p, sp) for p in PROMPTS]
            final = {}
            while eng.has_unfinished_requests():
                for o in eng.step():
                    if o.finished:
                        final[o.request_id] = (o.outputs[0].token_ids, o.outputs[0].logprobs)
            if saves and load_format == "auto" and tp > 1:
                eng.core.executor.save_sharded_state(shards)
            return [final[i] for i in ids]
        finally:
            eng.shutdown()
            pstate.destroy_model_parallel()

    one, two = run(ckpt, "auto", tp=1), run(ckpt, "auto")
    compare(one, two, 1e-2)                  # (sums in another order: the same few elements as above)
    if not saves:
        return
    again = run(shards, "sharded_state")
    assert [t for t, _ in again] == [t for t, _ in two]


@pytest.mark.parametrize("model", ["nemotron-tiny", "stablelm-tiny", "cohere-tiny", "phimoe-tiny", "glm4-moe-tiny", "granite-tiny", "arcee-tiny"])
def test_families_with_other_norms_and_experts(model):
    """Layers whose norm is not an RMS norm (it hands over no 8-bit rows), whose experts are routed in another way, or whose feed-forward
    is not gated run on the same projections."""
    def check(m):
        assert any(getattr(x, "mx_qw", None) is not None for x in m.modules())
    for tokens, logprobs in generate(model=model, quantization="mxfp4", load_format="dummy", check=check, tokens=2):
        assert len(tokens) == 2 and all(abs(v) < 1e4 for lp in logprobs for v in lp.values())
