"""Microscaled rows, norms, products and experts on the GPU against plain forms in 64 bits.

Tolerances.  Elements and scales of given numbers: equal.  A product's sum: the matrix instruction adds eight products at a time with 13
bits below the largest of them (each of the other seven may lose less than 2^-13 of it), everything else in 32 bits; so it is off by
at most 7 * 2^-13 < 2^-10 of the sum of the products' sizes, and a result in 16 bits by half a step more.  Over a whole result the losses,
of either sign, add up in squares: 2^-10 of the result's norm is six times what sums of many random products reach."""
import pytest
import torch

from tests import mx_oracle as oracle

pytestmark = pytest.mark.gpu
SUM = 2.0 ** -10
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(20)


def rows(m, k, dtype=torch.bfloat16, spread=0.7):
    x = torch.randn(m, k) * torch.exp(spread * torch.randn(k))
    return x.to(dtype)


def check_product(y, xv, wv, dtype, bias=None):
    """y against xv @ wv^T in 64 bits, element by element and as a whole."""
    want = xv @ wv.T
    if bias is not None:
        want = want + bias.double()
    size = xv.abs() @ wv.abs().T
    assert y.dtype == dtype and tuple(y.shape) == tuple(want.shape)
    off = (y.cpu().double() - want).abs()
    bound = SUM * size + HALF[dtype] * (want.abs() + SUM * size)
    if dtype == torch.float16:
        bound = bound + 2.0 ** -25                        # (half the smallest subnormal)
    assert (off <= bound).all(), f"worst {(off / bound).max():.3g} of the bound"
    if want.numel() > 256:
        assert off.norm() <= (SUM + HALF[dtype]) * want.norm()


# ------------------------------------------------------------------ rows
def hard_rows(dtype, width):
    """Blocks that go wrong easily: zeros of either sign, ties, largest values at and beside a scale's border, tiny and huge numbers."""
    x = torch.randn(40, width).double()
    for r, s in enumerate([448.0, 6.0, 448.0 * 2, 6.0 / 4, 464.0, 7.0, 1.75, 1.5]):
        x[r] = torch.rand(width).double() * s
        x[r, ::32] = s
        x[8 + r] = x[r]
        x[8 + r, ::32] = s * (1 + torch.finfo(dtype).eps)
    x[16] = 0
    x[17] = -0.0
    ties = torch.tensor(oracle.E2M1 + [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 2.5, -5.0, -0.25, 17 / 16, 19 / 16, -9 / 8, 1.0, 0.0]).repeat(2)
    x[18] = ties[:32].repeat(width // 32).double()
    x[19] = x[18] * 64
    tiny = float(torch.finfo(dtype).tiny)
    x[20] = x[18] * tiny
    x[21] = x[18] * tiny * torch.finfo(dtype).eps
    x[22] = torch.randn(width).double() * float(torch.finfo(dtype).max) / 8
    x[23, 0] = float(torch.finfo(dtype).max)
    x[24] = torch.randn(width).double() * 2.0 ** torch.randint(-30, 10, (width,)).double()
    return x.to(dtype)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,k", [(1, 32), (3, 96), (40, 128), (17, 2880), (257, 1024)])
def test_quantize(bits, dtype, m, k):
    from vllm_distributed_amd import ops
    x = hard_rows(dtype, k)[:m] if m == 40 else rows(m, k, dtype)
    r = ops.mx_quantize(x.cuda(), bits)
    code, byte, value = oracle.blocks(x, bits)
    assert torch.equal(r.s.view(torch.uint8).cpu().long(), byte)
    got = r.q.view(torch.uint8).cpu()
    assert torch.equal(got.long(), code) if bits == 8 else torch.equal(got, oracle.pack4(code))
    assert not r.payload.view(torch.uint8)[:, k * bits // 8:].any()                      # the padding is zeros
    assert torch.equal(ops.mx_dequantize(r, torch.float32).cpu().double(), value.float().double())


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantize_not_finite(bits, dtype):
    """A NaN or an infinity takes its block and no other."""
    from vllm_distributed_amd import ops
    x = rows(6, 128, dtype)
    x[0, 5], x[1, 40], x[2, 127], x[3, 0], x[3, 64] = float("nan"), float("inf"), float("-inf"), float("nan"), float("inf")
    r = ops.mx_quantize(x.cuda(), bits)
    _, byte, value = oracle.blocks(x, bits)
    assert torch.equal(r.s.view(torch.uint8).cpu().long(), byte) and (byte == 255).sum() == 5
    back = ops.mx_dequantize(r, torch.float32).cpu().double()
    assert torch.equal(back.isnan(), value.isnan()) and torch.equal(back.nan_to_num(), value.float().double().nan_to_num())


def test_quantize_strides_and_borders():
    """Rows of a wider matrix, of a transposed one, from an odd address; leading dimensions; no rows."""
    from vllm_distributed_amd import ops
    base = rows(24, 520).cuda()
    for x in (base[:, 8:8 + 256], base[::3, :96], base.t()[:96, :].t()[:, :96], base.flatten()[1:1 + 10 * 64].view(10, 64),
              base[:, 3:35]):
        r = ops.mx_quantize(x)
        code, byte, _ = oracle.blocks(x, 8)
        assert torch.equal(r.q.view(torch.uint8).cpu().long(), code) and torch.equal(r.s.view(torch.uint8).cpu().long(), byte)
    assert ops.mx_quantize(base.view(2, 12, 520)[:, :, :64]).shape == (24, 64)
    assert ops.mx_quantize(base[:0, :64]).shape == (0, 64)
    assert ops.mx_dequantize(ops.mx_quantize(base[:0, :64])).shape == (0, 64)


@pytest.mark.parametrize("at", range(8))
def test_one_row_of_any_stride(at):
    """One row that is a view: quantised, normed, multiplied, gated and through experts like its copy."""
    from tests.test_mx import one_row_views
    from vllm_distributed_amd import ops
    x = one_row_views(torch.bfloat16)[at]
    flat = x.reshape(1, 64).clone(memory_format=torch.contiguous_format)
    # (the same view of the same numbers on the device: a whole storage moves, strides and offset stay)
    base = torch.empty(0, dtype=x.dtype, device="cuda").set_(x.untyped_storage().cuda(), x.storage_offset(), x.shape, x.stride())
    assert base.stride() == x.stride() and torch.equal(base.cpu(), x)
    whole = flat.cuda()
    gain, residual = torch.ones(64, dtype=x.dtype).cuda(), rows(1, 64).cuda()
    w, _ = make(40, 64)
    w13, _ = make(256, 64, halves=2)
    e13, _ = make_experts(2, 256, 64, halves=2)
    e2, _ = make_experts(2, 64, 128)
    topi, topw = torch.tensor([[1, 0]], dtype=torch.int32).cuda(), torch.tensor([[0.75, 0.25]]).cuda()
    logits = torch.tensor([[0.5, -1.0]]).cuda()

    def bits(out):
        flat = [out] if isinstance(out, (torch.Tensor, ops.MxRows)) else list(out)
        parts = [t for o in flat for t in ((o.payload.view(torch.uint8), o.s.view(torch.uint8)) if isinstance(o, ops.MxRows) else (o,))]
        return [t.reshape(1, -1) for t in parts]
    calls = [lambda v: ops.mx_quantize(v, 8), lambda v: ops.mx_quantize(v, 4), lambda v: ops.rms_norm_mx(v, gain, 1e-5),
             lambda v: ops.fused_add_rms_norm_mx(v, residual, gain, 1e-5), lambda v: ops.mx_linear(v, w), lambda v: ops.mx_gate_up(v, w13)]
    if x.dim() == 2:
        calls += [lambda v: ops.mx_experts(v, topw, topi, e13, e2), lambda v: ops.mx_experts_routed(logits, v, 2, True, e13, e2)]
    for call in calls:
        assert all(torch.equal(a, b) for a, b in zip(bits(call(base)), bits(call(whole))))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_dequantize_every_code(dtype):
    from vllm_distributed_amd import ops
    table = torch.cat([oracle.TABLE[8], torch.tensor([float("nan")], dtype=torch.float64)])
    values = torch.cat([table, -table])
    q = torch.arange(256, dtype=torch.uint8).repeat(256, 1)
    byte = torch.arange(256, dtype=torch.uint8).unsqueeze(1).expand(256, 8).contiguous()
    r = ops.MxRows.of(q.cuda().view(torch.float8_e4m3fn), byte.cuda(), dtype)
    want = values.unsqueeze(0) * 2.0 ** (torch.arange(256).double() - 127).unsqueeze(1)
    want[255] = float("nan")
    got = ops.mx_dequantize(r).cpu()
    want = want.to(dtype)                             # (64 bits to 16: the values have four bits, so only subnormals round, once)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))


# ------------------------------------------------------------------ norms
def check_rows(r, v, slack):
    """8-bit rows against the numbers ``v [M, K]`` (64 bits) that they round, those being off by at most ``slack`` themselves: the scale is
    the power of two of a largest value within the slack, an element within half a step."""
    b, sl = v.reshape(v.shape[0], -1, 32), slack.reshape(v.shape[0], -1, 32)
    s = r.s.view(torch.uint8).cpu().long()
    limits = 448.0 * 2.0 ** torch.arange(-127, 128, dtype=torch.float64)
    lo = torch.searchsorted(limits, (b.abs() - sl).clamp_min(0).amax(-1).contiguous())
    hi = torch.searchsorted(limits, (b.abs() + sl).amax(-1).contiguous())
    assert ((lo <= s) & (s <= hi)).all()
    scale = (2.0 ** (s.double() - 127)).unsqueeze(-1)
    got = r.q.cpu().double().reshape(b.shape) * scale
    bound = sl + torch.maximum(2.0 ** -4 * (b.abs() + sl), 2.0 ** -10 * scale)
    off = (got - b).abs()
    assert (off <= bound).all(), f"worst {(off / bound).max():.3g} of the bound"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,h", [(1, 32), (1, 4096), (3, 96), (130, 2880), (7, 8192), (2, 32768), (64, 5120)])
@pytest.mark.parametrize("form", ["plain", "residual", "slabs"])
def test_norm(dtype, m, h, form):
    from vllm_distributed_amd import ops
    x, gain = rows(m, h, dtype), (1 + 0.2 * torch.randn(h)).to(dtype)
    residual = (4 * torch.randn(m, h)).to(dtype)
    if form == "plain":
        r, out, total = ops.rms_norm_mx(x.cuda(), gain.cuda(), 1e-5), None, x.double()
    elif form == "residual":
        r, out = ops.fused_add_rms_norm_mx(x.cuda(), residual.cuda(), gain.cuda(), 1e-5)
        total = x.double() + residual.double()
    else:
        slabs = torch.randn(3, m, h)
        r, out = ops.reduce_add_rms_norm_mx(slabs.cuda(), residual.cuda(), gain.cuda(), 1e-5)
        total = slabs.double().sum(0) + residual.double()
    if out is not None:
        # (one rounding of a 32-bit sum of up to four numbers, whose own roundings may carry it over a border)
        half = HALF[dtype] * total.abs() + (2.0 ** -25 if dtype == torch.float16 else 0)
        sums = 0 if form == "residual" else 4 * 2.0 ** -24 * (slabs.double().abs().sum(0) + residual.double().abs())
        assert ((out.cpu().double() - total).abs() <= half + 2 * sums).all()
    v = total / torch.sqrt((total ** 2).mean(-1, keepdim=True) + 1e-5) * gain.double()
    # 32-bit arithmetic: a sum of h squares in at most 10 + log2(1024) dependent additions, root, division, two products, each 2^-24
    size = (slabs.double().abs().sum(0) + residual.double().abs()) / total.abs().clamp_min(1e-30) if form == "slabs" else torch.ones_like(v)
    check_rows(r, v, (40 + 4 * size) * 2.0 ** -24 * v.abs())
    assert not r.payload.view(torch.uint8)[:, h:].any()


def test_norm_keeps_its_inputs_and_takes_strides():
    from vllm_distributed_amd import ops
    wide = rows(9, 1024).cuda()
    x, residual, gain = wide[:, 128:640], rows(9, 512).cuda(), torch.ones(512, dtype=torch.bfloat16).cuda()
    before = wide.clone(), residual.clone()
    r, out = ops.fused_add_rms_norm_mx(x, residual, gain, 1e-6)
    assert torch.equal(wide, before[0]) and torch.equal(residual, before[1])
    again, out2 = ops.fused_add_rms_norm_mx(x.contiguous(), residual, gain, 1e-6)
    assert torch.equal(r.payload.view(torch.uint8), again.payload.view(torch.uint8)) and torch.equal(r.s.view(torch.uint8), again.s.view(torch.uint8)) and torch.equal(out, out2)


@pytest.mark.parametrize("at", [1, 4, 8])
def test_norm_of_a_residual_from_any_address(at):
    from vllm_distributed_amd import ops
    m, h = 3, 96
    flat = rows(1, (m + 1) * h).flatten().cuda()
    x, residual, gain = rows(m, h).cuda(), flat[at:at + m * h].view(m, h), (1 + 0.2 * torch.randn(h)).to(torch.bfloat16).cuda()
    slabs = torch.randn(2, m, h).cuda()
    before = flat.clone()
    for call in (lambda r: ops.fused_add_rms_norm_mx(x, r, gain, 1e-5), lambda r: ops.reduce_add_rms_norm_mx(slabs, r, gain, 1e-5)):
        (a, sa), (b, sb) = call(residual), call(residual.clone())
        assert torch.equal(sa, sb) and torch.equal(a.payload.view(torch.uint8), b.payload.view(torch.uint8))
        assert torch.equal(a.s.view(torch.uint8), b.s.view(torch.uint8)) and torch.equal(flat, before)


# ------------------------------------------------------------------ products
def make(n, k, halves=1, spread=3):
    from vllm_distributed_amd.ops import quant
    gen = torch.Generator().manual_seed(n * 7 + k)
    packed, byte, v = oracle.random_weight(n, k, gen, spread)
    return quant.pack_mx(packed.cuda(), byte.cuda(), halves=halves), v


@pytest.mark.parametrize("n,k", [(8, 32), (40, 96), (264, 160), (1000, 1056), (512, 2880), (4096, 512), (96, 14336)])
@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 33, 65, 130])
def test_linear(m, n, k):
    from vllm_distributed_amd import ops
    dtype = torch.float16 if (m + n) % 3 == 0 else torch.bfloat16
    x = (rows(m, k).float() / 8).to(dtype)
    w, wv = make(n, k, spread=1)
    bias = torch.randn(n).to(dtype) if m % 2 else None
    y = ops.mx_linear(x.cuda(), w, None if bias is None else bias.cuda())
    check_product(y, oracle.blocks(x, 8)[2], wv, dtype, bias)


@pytest.mark.parametrize("m,n,k", [(300, 328, 640), (513, 1288, 384), (1024, 256, 128), (700, 4096, 1056), (2049, 520, 288)])
def test_linear_many_rows(m, n, k):
    from vllm_distributed_amd import ops
    x = rows(m, k)
    w, wv = make(n, k)
    check_product(ops.mx_linear(x.cuda(), w), oracle.blocks(x, 8)[2], wv, torch.bfloat16)


@pytest.mark.parametrize("m", [1, 20, 400])
def test_linear_of_every_scale(m):
    """Scales over their whole range on both sides, the products staying within 32 bits."""
    from vllm_distributed_amd import ops
    from vllm_distributed_amd.ops import quant
    n, k = 48, 512
    gen = torch.Generator().manual_seed(3)
    packed, _, _ = oracle.random_weight(n, k, gen)
    e = torch.randint(-100, 101, (k // 32,), generator=gen)
    wb = (127 + e).expand(n, -1).to(torch.uint8).contiguous()
    x = torch.randn(m, k) * (2.0 ** -e.float()).repeat_interleave(32)
    r = ops.mx_quantize(x.cuda(), 8)
    r.dtype = torch.bfloat16
    code = torch.stack([packed & 15, packed >> 4], -1).reshape(n, k).long()
    wv = oracle.TABLE[4][code & 7] * torch.where(code > 7, -1.0, 1.0).double() * (2.0 ** e.double()).repeat_interleave(32)
    check_product(ops.mx_linear(r, quant.pack_mx(packed.cuda(), wb.cuda())), oracle.blocks(x, 8)[2], wv, torch.bfloat16)


@pytest.mark.parametrize("m", [3, 40, 300])
def test_linear_rows_do_not_mix(m):
    """A NaN makes its row NaN and leaves every other row's bits as they were; so does a NaN scale of the weight with its column."""
    from vllm_distributed_amd import ops
    x = rows(m, 640)
    w, _ = make(136, 640)
    clean = ops.mx_linear(x.cuda(), w)
    bad = x.clone()
    bad[m // 2, 77] = float("nan")
    y = ops.mx_linear(bad.cuda(), w)
    keep = torch.arange(m) != m // 2
    assert y[m // 2].isnan().all() and torch.equal(y[keep.cuda()], clean[keep.cuda()])
    ws = w.ws.clone()
    ws[2, 0, 5, 1] = 255                                  # row 37, columns 128 .. 159
    y = ops.mx_linear(x.cuda(), ops.MxWeight(w.qw, ws, w.rows))
    cols = torch.arange(136) != 37
    assert y[:, 37].isnan().all() and torch.equal(y[:, cols.cuda()], clean[:, cols.cuda()])


@pytest.mark.parametrize("mt,nt,ksplit", [(2, 2, 1), (2, 2, 2), (4, 2, 1), (4, 2, 3), (8, 4, 1), (8, 4, 3), (2, 4, 1)])
@pytest.mark.parametrize("m,n,k", [(1, 8, 544), (130, 1000, 544), (257, 264, 2880), (700, 2560, 1184)])
def test_every_shape_of_the_ring(m, n, k, mt, nt, ksplit, monkeypatch):
    """Shapes of the launch that the plan keeps for other sizes, at ragged ones: the answer is the same."""
    from vllm_distributed_amd import ops
    from vllm_distributed_amd.ops import hip
    x, b = rows(m, k), torch.randn(n).to(torch.bfloat16)
    w, wv = make(n, k)
    xr = ops.mx_quantize(x.cuda())
    monkeypatch.setattr(hip, "mx_plan", lambda *a: (hip._mx_shape(mt, nt, 1), ksplit))
    if mt == 8 or nt == 2:
        check_product(ops.mx_linear(xr, w, b.cuda()), oracle.blocks(x, 8)[2], wv, torch.bfloat16, b)
    if nt == 4 and ksplit == 1:
        w, wv = make(256 * (n // 256 + 1), k, halves=2, spread=1)
        xr = ops.mx_quantize((x.float() / k ** 0.5).to(torch.bfloat16).cuda())
        v, slack = gated_slack(ops.mx_dequantize(xr, torch.float32).cpu().double(), wv, None, 0.0)
        check_rows(ops.mx_gate_up(xr, w), v, slack)


BIG_TILES = [(1, 8, 32), (255, 264, 128), (256, 256, 1056), (257, 1000, 160), (2049, 2568, 384), (300, 1000, 1184), (2049, 9992, 288)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k", BIG_TILES)
def test_large_tiles(m, n, k, dtype, monkeypatch):
    """The kernel of 256-row tiles at rows, columns and steps that leave parts of a tile empty: one step, an odd number of them, columns of one
    die alone, and (the last) more tiles than workgroups, so that loads run on into the next one."""
    from vllm_distributed_amd import ops
    from vllm_distributed_amd.ops import hip
    monkeypatch.setattr(hip, "mx_plan", lambda *a: (hip.MX_BIG, 1))
    x = (rows(m, k).float() / 8).to(dtype)
    w, wv = make(n, k, spread=1)
    bias = torch.randn(n).to(dtype)
    xr, xv = ops.mx_quantize(x.cuda()), oracle.blocks(x, 8)[2]
    check_product(ops.mx_linear(xr, w, bias.cuda()), xv, wv, dtype, bias)
    check_product(ops.mx_linear(xr, w), xv, wv, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,inter,k,limit", [(1, 128, 32, 0.0), (255, 384, 160, 7.0), (513, 1408, 288, 0.0), (2049, 256, 128, 7.0),
                                             (300, 128, 1184, 0.0), (2049, 3200, 288, 7.0)])
def test_gated_large_tiles(m, inter, k, limit, dtype, monkeypatch):
    """Likewise the gated product, whose tiles have columns of both halves."""
    from vllm_distributed_amd import ops
    from vllm_distributed_amd.ops import hip
    monkeypatch.setattr(hip, "mx_plan", lambda *a: (hip.MX_BIG, 1))
    x = (rows(m, k, spread=0.3).float() / k ** 0.5).to(dtype)
    w, wv = make(2 * inter, k, halves=2, spread=1)
    bias = torch.randn(2 * inter).to(dtype)
    for b in (bias, None):
        r = ops.mx_gate_up(ops.mx_quantize(x.cuda()), w, None if b is None else b.cuda(), limit=limit)
        check_rows(r, *gated_slack(oracle.blocks(x, 8)[2], wv, b, limit))


@pytest.mark.parametrize("mt,nt,ksplit", [(2, 2, 2), (4, 2, 3), (8, 4, 2), (8, 4, 3)])
@pytest.mark.parametrize("m,inter,k,limit", [(33, 256, 1056, 0.0), (130, 640, 544, 7.0)])
def test_gated_products_of_a_split_reduction(m, inter, k, limit, mt, nt, ksplit, monkeypatch):
    from vllm_distributed_amd import ops
    from vllm_distributed_amd.ops import hip
    monkeypatch.setattr(hip, "mx_plan", lambda *a: (hip._mx_shape(mt, nt, 1), ksplit))
    x = (rows(m, k, spread=0.3).float() / k ** 0.5).to(torch.bfloat16)
    w, wv = make(2 * inter, k, halves=2, spread=1)
    b = torch.randn(2 * inter).to(torch.bfloat16)
    check_rows(ops.mx_gate_up(x.cuda(), w, b.cuda(), limit=limit), *gated_slack(oracle.blocks(x, 8)[2], wv, b, limit))


@pytest.mark.parametrize("m,n,k,gated,shape", [
    (2, 1000, 288, False, (1, 1, 8)), (7, 1000, 288, False, (1, 1, 8)), (3, 4104, 160, False, (1, 2, 8)), (13, 4104, 160, False, (1, 2, 8)),
    (2, 16424, 160, False, (1, 2, 8)), (3, 16424, 160, False, (1, 4, 4)), (9, 16424, 160, False, (1, 4, 4)), (4, 64, 11520, False, (1, 1, 8)),
    (1, 512, 288, True, (1, 4, 8)), (11, 512, 288, True, (1, 4, 8)), (4, 256, 11520, True, (1, 4, 8)), (4, 16384, 160, True, (1, 4, 4)),
    (12, 16384, 160, True, (1, 4, 4))])
def test_every_shape_of_the_stream(m, n, k, gated, shape):
    """Every launch of the streaming kernel that the plan makes, at sizes where it makes it: up to four rows are quantised inside (11520
    columns: as many as fit, next to the sums of eight waves), others in front."""
    from vllm_distributed_amd import ops
    from vllm_distributed_amd.ops import hip
    kb = (k + 127) // 128
    assert hip.mx_plan(m, n, kb, True, gated) == (hip._mx_shape(*shape), 1) and hip.mx_fused_ok(m, kb) == (m <= 4)
    x = (rows(m, k, spread=0.3).float() / k ** 0.5).to(torch.bfloat16)
    w, wv = make(n, k, halves=2 if gated else 1, spread=1)
    b = torch.randn(n).to(torch.bfloat16)
    xv = oracle.blocks(x, 8)[2]
    for bias in (b, None):
        on_gpu = None if bias is None else bias.cuda()
        if gated:
            check_rows(ops.mx_gate_up(x.cuda(), w, on_gpu), *gated_slack(xv, wv, bias, 0.0))
        else:
            check_product(ops.mx_linear(x.cuda(), w, on_gpu), xv, wv, torch.bfloat16, bias)


@pytest.mark.parametrize("m", [17, 40, 130])
def test_operands_past_32_bit_offsets_stream(m, monkeypatch):
    """What runs for operands of 4 GiB and more, at small ones."""
    from vllm_distributed_amd import ops
    from vllm_distributed_amd.ops import hip
    monkeypatch.setattr(hip, "mx_big_ok", lambda *a: False)
    monkeypatch.setattr(hip, "mx_sorted_ok", lambda *a: False)
    x = (rows(m, 1056).float() / 32).to(torch.bfloat16)
    w, wv = make(264, 1056)
    check_product(ops.mx_linear(x.cuda(), w), oracle.blocks(x, 8)[2], wv, torch.bfloat16)
    w, wv = make(512, 1056, halves=2, spread=1)
    v, slack = gated_slack(oracle.blocks(x, 8)[2], wv, None, 0.0)
    check_rows(ops.mx_gate_up(x.cuda(), w), v, slack)
    w13, v13 = make_experts(2, 256, 1056, halves=2)
    w2, v2 = make_experts(2, 96, 128)
    topi = torch.stack([torch.randperm(2) for _ in range(m)]).int()
    topw = torch.rand(m, 2)
    y = ops.mx_experts(x.cuda(), topw.cuda(), topi.cuda(), w13, w2)
    want, bound = expert_block(oracle.blocks(x, 8)[2], topw, topi, v13, v2, None, None, 0.0)
    assert ((y.cpu().double() - want).abs() <= bound).all()


def test_rows_of_4_gib():
    """530 000 rows of 8192: payload past 32-bit offsets.  Rows from both ends and the middle."""
    from vllm_distributed_amd import ops
    m, k = 530_000, 8192
    some = torch.tensor([0, 1, 262_143, 262_144, 524_287, 524_288, m - 1])
    seven = rows(7, k)
    x = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")
    x[some.cuda()] = seven.cuda()
    w, wv = make(24, k)
    r = ops.mx_quantize(x)
    del x
    y = ops.mx_linear(r, w)
    check_product(y[some.cuda()], oracle.blocks(seven, 8)[2], wv, torch.bfloat16)
    y[some.cuda()] = 0
    assert not y.any()
    back = ops.mx_dequantize(ops.MxRows(r.payload[-2:], r.scales[-2:], k, 8, r.dtype), torch.float32)
    assert torch.equal(back[1].cpu().double(), oracle.blocks(seven, 8)[2][6])


@pytest.mark.parametrize("m", [2, 40])
def test_weight_of_4_gib(m):
    """1 056 000 columns of 8192: the weight's tiles past 32-bit offsets.  Columns from both ends and beside the border."""
    from vllm_distributed_amd import ops
    from vllm_distributed_amd.ops import quant
    n, k = 1_056_000, 8192
    q, s, wv = oracle.random_weight(48, k, torch.Generator().manual_seed(m), 1)
    part = quant.pack_mx(q.cuda(), s.cuda())
    w = ops.MxWeight(torch.zeros(n // 16, k // 128, 64, 4, dtype=torch.int32, device="cuda"),
                     torch.zeros(n // 16, k // 512, 64, 4, dtype=torch.uint8, device="cuda"), n)
    at = [0, 65_536, n // 16 - 1]
    for i, t in enumerate(at):
        w.qw[t], w.ws[t] = part.qw[i], part.ws[i]
    x = rows(m, k, spread=0.3)
    y = ops.mx_linear(x.cuda(), w)
    for i, t in enumerate(at):
        check_product(y[:, 16 * t:16 * t + 16], oracle.blocks(x, 8)[2], wv[16 * i:16 * i + 16], torch.bfloat16)
        y[:, 16 * t:16 * t + 16] = 0
    assert not y.any()


@pytest.mark.parametrize("m,n,k", [(40, 512, 4096), (64, 2880, 4096)])
def test_partials_and_the_norm_behind_them(m, n, k):
    from vllm_distributed_amd import ops
    x, residual, gain = rows(m, k), rows(m, n), (1 + 0.1 * torch.randn(n)).to(torch.bfloat16)
    w, wv = make(n, k)
    xr = ops.mx_quantize(x.cuda())
    slabs = ops.mx_linear_partials(xr, w)
    assert slabs is not None and slabs.dtype == torch.float32 and slabs.shape[1:] == (m, n)
    xv = oracle.blocks(x, 8)[2]
    size = xv.abs() @ wv.abs().T
    assert ((slabs.double().sum(0).cpu() - xv @ wv.T).abs() <= SUM * size).all()
    r, out = ops.reduce_add_rms_norm_mx(slabs, residual.cuda(), gain.cuda(), 1e-5)
    total = slabs.double().sum(0).cpu() + residual.double()
    v = total / torch.sqrt((total ** 2).mean(-1, keepdim=True) + 1e-5) * gain.double()
    sums = (slabs.double().abs().sum(0).cpu() + residual.double().abs()) / total.abs().clamp_min(1e-30)
    check_rows(r, v, (40 + (slabs.shape[0] + 1) * sums) * 2.0 ** -24 * v.abs())


# ------------------------------------------------------------------ gated products
def gated_slack(xv, wv, bias, limit, alpha=1.702):
    """(the activation in 64 bits, how far sums within their bound may move it)."""
    h = xv @ wv.T
    h = h if bias is None else h + bias.double()
    d = 1.01 * SUM * (xv.abs() @ wv.abs().T)
    v = oracle.gated(h, limit, alpha)
    g, u = h.chunk(2, -1)
    dg, du = d.chunk(2, -1)
    # |d silu / dg| <= 1.1, of g sigmoid(alpha g) too; sigmoid by exp2 and a reciprocal of 1 ulp each: 2^-21 of the result
    f = (g.clamp(max=limit) if limit else g).abs()
    up = (u.clamp(-limit, limit) + 1).abs() if limit else u.abs()
    return v, 1.1 * dg * (up + du) + f * du + 2.0 ** -20 * v.abs() + 1e-30


@pytest.mark.parametrize("m", [1, 16, 19, 64, 100, 300, 777])
@pytest.mark.parametrize("inter,k,limit,bias", [(128, 128, 0.0, False), (256, 288, 7.0, True), (640, 1120, 0.0, True), (128, 4096, 7.0, False)])
def test_gate_up(m, inter, k, limit, bias):
    from vllm_distributed_amd import ops
    x = (rows(m, k, spread=0.3).float() / k ** 0.5).to(torch.bfloat16)
    w, wv = make(2 * inter, k, halves=2, spread=1)
    b = torch.randn(2 * inter).to(torch.bfloat16) if bias else None
    r = ops.mx_gate_up(x.cuda(), w, None if b is None else b.cuda(), limit=limit)
    assert r.shape == (m, inter)
    v, slack = gated_slack(oracle.blocks(x, 8)[2], wv, b, limit)
    check_rows(r, v, slack)


def test_feed_forward_of_rows():
    """Norm, gate and up, down: what a decoder layer runs, against the same in 64 bits over the rows that each step left."""
    from vllm_distributed_amd import ops
    m, h, inter = 37, 512, 1024
    x, residual, gain = rows(m, h), rows(m, h), torch.ones(h, dtype=torch.bfloat16)
    w13, v13 = make(2 * inter, h, halves=2, spread=1)
    w2, v2 = make(h, inter, spread=1)
    r, out = ops.fused_add_rms_norm_mx(x.cuda(), residual.cuda(), gain.cuda(), 1e-5)
    a = ops.mx_gate_up(r, w13)
    v, slack = gated_slack(ops.mx_dequantize(r, torch.float32).cpu().double(), v13, None, 0.0)
    check_rows(a, v, slack)
    check_product(ops.mx_linear(a, w2), ops.mx_dequantize(a, torch.float32).cpu().double(), v2, torch.bfloat16)


# ------------------------------------------------------------------ experts
def make_experts(e, n, k, halves=1):
    from vllm_distributed_amd.ops import quant
    gen = torch.Generator().manual_seed(e * 31 + n + k)
    parts = [oracle.random_weight(n, k, gen, 1) for _ in range(e)]
    w = quant.pack_mx(torch.stack([p[0] for p in parts]).cuda(), torch.stack([p[1] for p in parts]).cuda(), halves=halves)
    return w, torch.stack([p[2] for p in parts])


def expert_block(xv, topw, topi, v13, v2, b13, b2, limit):
    """The sparse block of rows ``xv`` in 64 bits (matrices as numbers, ``[E, ..]``), and how far a bfloat16 result may be from it."""
    want = torch.zeros(xv.shape[0], v2.shape[1], dtype=torch.float64)
    bound = torch.zeros_like(want)
    for j in range(len(v2)):
        r, c = (topi == j).nonzero(as_tuple=True)
        if not len(r):
            continue
        v, slack = gated_slack(xv[r], v13[j], None if b13 is None else b13[j].cpu(), limit)
        a = oracle.blocks(v, 8)[2]
        z = a @ v2[j].T + (0 if b2 is None else b2[j].cpu().double())
        # an activation beside the middle of two elements may go to the other: a step of 2^-3 of it (2^-9 of its scale where subnormal)
        flips = torch.maximum(2.0 ** -3 * v.abs(), 2.0 ** -18 * v.abs().reshape(len(r), -1, 32).amax(-1).repeat_interleave(32, 1)) + slack
        near = oracle.blocks(v + slack, 8)[2] != oracle.blocks(v - slack, 8)[2]
        d = (flips * near) @ v2[j].abs().T + SUM * (a.abs() @ v2[j].abs().T)
        want.index_add_(0, r, z * topw[r, c].double().unsqueeze(1))
        bound.index_add_(0, r, (d + 2.0 ** -20 * z.abs()) * topw[r, c].double().unsqueeze(1))      # (up to four 32-bit products and sums)
    return want, bound + 2.0 ** -8 * (want.abs() + bound)


@pytest.mark.parametrize("t,e,k,h,inter,limit", [(1, 8, 2, 128, 128, 0.0), (16, 128, 4, 288, 160, 7.0), (9, 4, 4, 160, 128, 7.0),
                                                 (64, 4, 2, 416, 160, 7.0), (200, 4, 2, 160, 288, 7.0), (220, 4, 2, 288, 160, 0.0),
                                                 (70, 8, 2, 256, 384, 0.0), (40, 4, 2, 416, 160, 7.0), (150, 4, 2, 160, 288, 7.0), (300, 5, 3, 96, 96, 7.0), (1200, 4, 2, 256, 128, 0.0), (513, 3, 2, 160, 416, 7.0)])
def test_experts(t, e, k, h, inter, limit):
    from vllm_distributed_amd import ops
    from vllm_distributed_amd.ops import quant
    x = (rows(t, h, spread=0.3).float() / h ** 0.5).to(torch.bfloat16)
    w13, v13 = make_experts(e, 2 * inter, h, halves=2)
    w2, v2 = make_experts(e, h, inter)
    b13 = torch.randn(e, 2 * inter).to(torch.bfloat16) if limit else None
    b2 = torch.randn(e, h).to(torch.bfloat16) if limit else None
    topi = torch.stack([torch.randperm(e)[:k] for _ in range(t)]).int()
    topi[topi == e - 1] = 0                              # an expert that nobody chose, one that a row chose twice
    topw = torch.rand(t, k)
    y = ops.mx_experts(x.cuda(), topw.cuda(), topi.cuda(), w13, w2, None if b13 is None else quant.pad_mx_bias(b13, 2).cuda(),
                       None if b2 is None else b2.cuda(), limit=limit)
    want, bound = expert_block(oracle.blocks(x, 8)[2], topw, topi, v13, v2, b13, b2, limit)
    off = (y.cpu().double() - want).abs()
    assert (off <= bound).all(), f"worst {(off / bound).max():.3g} of the bound"
    assert off.norm() <= 2.0 ** -6 * want.norm()


def test_experts_of_more_outputs_than_workgroups():
    """256-row tiles, 24 of them by 11 columns: loads run on from one expert's output into the next one's."""
    from vllm_distributed_amd import ops
    from vllm_distributed_amd.ops import hip
    t, e, k, h, inter = 2800, 8, 2, 160, 1408
    assert hip.mx_tile_rows(t * k, e) == 256
    x = (rows(t, h, spread=0.3).float() / h ** 0.5).to(torch.bfloat16)
    w13, v13 = make_experts(e, 2 * inter, h, halves=2)
    w2, v2 = make_experts(e, h, inter)
    topi = torch.stack([torch.randperm(e)[:k] for _ in range(t)]).int()
    topw = torch.rand(t, k)
    y = ops.mx_experts(x.cuda(), topw.cuda(), topi.cuda(), w13, w2)
    want, bound = expert_block(oracle.blocks(x, 8)[2], topw, topi, v13, v2, None, None, 0.0)
    off = (y.cpu().double() - want).abs()
    assert (off <= bound).all(), f"worst {(off / bound).max():.3g} of the bound"
    assert off.norm() <= 2.0 ** -6 * want.norm()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t", [1, 7, 16, 17, 300])
@pytest.mark.parametrize("e,k", [(8, 2), (64, 6), (3, 3)])
def test_experts_behind_their_router(t, e, k, dtype):
    """The same bits as the choice and the experts in calls of their own, whole and in two ranks' halves."""
    from vllm_distributed_amd import ops
    h, inter = 160, 128
    x = (rows(t, h, spread=0.3).float() / h ** 0.5).to(dtype).cuda()
    w13, _ = make_experts(e, 2 * inter, h, halves=2)
    w2, _ = make_experts(e, h, inter)
    b2 = torch.randn(e, h).to(dtype).cuda()
    for logits in (torch.randn(t, e).cuda(), torch.randn(t, e).to(dtype).cuda()):
        topw, topi = ops.moe_topk(logits, k, True)
        want = ops.mx_experts(x, topw, topi, w13, w2, None, b2, limit=7.0)
        assert torch.equal(ops.mx_experts_routed(logits, x, k, True, w13, w2, None, b2, limit=7.0), want)
        part = lambda w, lo, n: ops.MxWeight(w.qw[lo:lo + n].contiguous(), w.ws[lo:lo + n].contiguous(), w.rows)
        for lo, n in ((0, e // 2), (e // 2, e - e // 2)):
            args = part(w13, lo, n), part(w2, lo, n), None, b2[lo:lo + n].contiguous(), lo, n
            assert torch.equal(ops.mx_experts_routed(logits, x, k, True, *args), ops.mx_experts(x, topw, topi, *args, e))
    with pytest.raises(ValueError):
        ops.mx_experts_routed(torch.randn(t, e + 1).cuda(), x, k, True, w13, w2)


@pytest.mark.parametrize("t", [3, 40, 200, 600])
def test_experts_nobody_has(t):
    """Slots of numbers that are no expert's add nothing, at each kind of tile; no rows are none."""
    from vllm_distributed_amd import ops
    e, k, h, inter = 4, 3, 96, 160
    x = (rows(t, h, spread=0.3).float() / h ** 0.5).to(torch.bfloat16)
    w13, v13 = make_experts(e, 2 * inter, h, halves=2)
    w2, v2 = make_experts(e, h, inter)
    topi = torch.stack([torch.randperm(e)[:k] for _ in range(t)]).int()
    topi[::2, 1], topi[1::3, 2], topi[0] = -1, e + 5, -7
    topw = torch.rand(t, k)
    want, bound = expert_block(oracle.blocks(x, 8)[2], topw, topi, v13, v2, None, None, 0.0)
    for rows_ in (x.cuda(), ops.mx_quantize(x.cuda())):
        y = ops.mx_experts(rows_, topw.cuda(), topi.cuda(), w13, w2)
        assert ((y.cpu().double() - want).abs() <= bound).all() and not y[0].any()
    assert ops.mx_experts(x[:0].cuda(), topw[:0].cuda(), topi[:0].cuda(), w13, w2).shape == (0, h)


@pytest.mark.parametrize("t", [5, 33, 700])
def test_experts_of_two_ranks_add_up(t):
    """Expert parallel: each rank adds its experts' part; in one row's 32-bit sum the parts are those of the whole block."""
    from vllm_distributed_amd import ops
    e, k, h, inter = 6, 3, 128, 128
    x = rows(t, h, spread=0.3).cuda()
    w13, _ = make_experts(e, 2 * inter, h, halves=2)
    w2, _ = make_experts(e, h, inter)
    topi = torch.stack([torch.randperm(e)[:k] for _ in range(t)]).int().cuda()
    topw = torch.rand(t, k).cuda()
    whole = ops.mx_experts(x, topw, topi, w13, w2)
    assert torch.equal(ops.mx_experts(ops.mx_quantize(x), topw, topi, w13, w2), whole)      # (rows that are 8-bit already)
    parts = []
    for lo in (0, 3):
        sl = lambda w: ops.MxWeight(w.qw[lo:lo + 3].contiguous(), w.ws[lo:lo + 3].contiguous(), w.rows)  # noqa: E731
        parts.append(ops.mx_experts(x, topw, topi, sl(w13), sl(w2), expert_start=lo, local_experts=3, num_experts=e))
    got, want = (parts[0].double() + parts[1].double()), whole.double()
    # each rounds a 32-bit sum once, of numbers up to some size s: half a step of each part and of the whole, 2^-20 s in the sums
    assert ((got - want).abs() <= (2.0 ** -8 + 2.0 ** -12) * (parts[0].double().abs() + parts[1].double().abs() + want.abs())).all()


# ------------------------------------------------------------------ how they are used
def test_graph_replays_and_streams():
    """A captured norm, gate and up, down and experts over changed inputs, replayed with eager work between; the same on another stream."""
    from vllm_distributed_amd import ops
    m, h, inter = 20, 256, 384
    w13, _ = make(2 * inter, h, halves=2)
    w2, _ = make(h, inter)
    e13, _ = make_experts(4, 2 * inter, h, halves=2)
    e2, _ = make_experts(4, h, inter)
    gain = torch.ones(h, dtype=torch.bfloat16).cuda()
    x, residual = rows(m, h).cuda(), rows(m, h).cuda()
    topi = torch.randint(0, 4, (m, 2), dtype=torch.int32).cuda()
    topw = torch.rand(m, 2).cuda()

    def step():
        r, res = ops.fused_add_rms_norm_mx(x, residual, gain, 1e-5)
        y = ops.mx_linear(ops.mx_gate_up(r, w13), w2)
        return y, res, ops.mx_experts(r, topw, topi, e13, e2), ops.mx_dequantize(ops.mx_quantize(x, 4))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, step()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        x.copy_(rows(m, h))
        topi.copy_(torch.randint(0, 4, (m, 2), dtype=torch.int32))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i


def test_refusals():
    from vllm_distributed_amd import ops
    from vllm_distributed_amd.ops import quant
    x = rows(4, 128).cuda()
    w, _ = make(64, 128)
    with pytest.raises(ValueError):
        ops.mx_linear(rows(4, 256).cuda(), w)
    with pytest.raises(ValueError):
        ops.mx_linear(ops.mx_quantize(x, 4), w)
    with pytest.raises(ValueError):
        ops.mx_gate_up(x, w)
    with pytest.raises(AssertionError):
        ops.mx_linear(x, w, torch.zeros(63, dtype=torch.bfloat16).cuda())
    with pytest.raises(AssertionError):
        ops.mx_linear(x, ops.MxWeight(w.qw, w.ws[:-1], w.rows))
    with pytest.raises(ValueError):
        ops.mx_linear(x, ops.MxWeight(w.qw.cpu(), w.ws.cpu(), w.rows))
    with pytest.raises(ValueError):
        quant.pack_mx(torch.zeros(12, 64, dtype=torch.uint8), torch.zeros(12, 4, dtype=torch.uint8))
