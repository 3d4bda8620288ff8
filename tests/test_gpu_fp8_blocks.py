"""8-bit blocks on the GPU: quantise / dequantise bit for bit, the checkpointed activation and its
gradient, the block-scaled matrix product, and a feed-forward step that uses them together."""
from __future__ import annotations

import math

import pytest
import torch

import fp8_reference as R
import hc

pytestmark = pytest.mark.gpu

KINDS = ["f32", "f16", "bf16"]
F8 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops(cuda):
    return hc.load_torch_ops()


def rnd(shape, seed, kind="f32", scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * scale
    if len(shape) and shape[-1] > 3:
        x[..., 3] *= 20  # a large channel
    return x.to(R.DTYPES[kind])


def same_codes(q, ref_values, what):
    assert torch.equal(q.float().cpu(), ref_values), what


# ------------------------------------------------------------------------------ quantise
ROW_SHAPES = [(1, 1), (1, 128), (3, 127), (2, 129), (5, 8), (7, 256), (4, 1000), (3, 1001), (2, 3, 264), (130, 384),
              (1, 8192), (1025, 136)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", ROW_SHAPES, ids=str)
def test_quantize_rows(cuda, shape, kind):
    x = rnd(shape, 1, kind)
    q, scale = hc.quantize_fp8_block(x.cuda())
    ref_q, ref_s = R.quantize_rows(x)
    assert torch.equal(scale.cpu(), ref_s)
    same_codes(q, ref_q, "codes")
    back = hc.dequantize_fp8_block(q, scale, torch.float32)
    spread = ref_s.repeat_interleave(128, -1)[..., : shape[-1]]
    assert torch.equal(back.cpu(), ref_q * spread)  # one fp32 product
    for dt in (torch.float16, torch.bfloat16):
        assert torch.equal(hc.dequantize_fp8_block(q, scale, dt).cpu(), (ref_q * spread).to(dt))
    # an element is off by half a code step, or by half the smallest code step times the scale
    err = (back.cpu().double() - x.double()).abs()
    assert bool((err <= x.double().abs() * 2.0**-4 * (1 + 4 * R.U) + spread.double() * 2.0**-10 * (1 + 4 * R.U)).all())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", [(1, 1), (128, 128), (129, 127), (300, 260), (7, 1000), (256, 384)], ids=str)
def test_quantize_tiles(cuda, shape, kind):
    x = rnd(shape, 2, kind)
    q, scale = hc.quantize_fp8_block(x.cuda(), 128)
    ref_q, ref_s = R.quantize_tiles(x)
    assert torch.equal(scale.cpu(), ref_s)
    same_codes(q, ref_q, "codes")
    back = hc.dequantize_fp8_block(q, scale, torch.float32, 128)
    assert torch.equal(back.cpu(), (ref_q.double() * R.spread(ref_s, shape, 128)).float())


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_extremes(cuda, block_rows):
    """Zero, subnormal, tiny, huge and non-finite blocks."""
    x = torch.zeros(5 * 128, 128)
    x[128, 5] = 1e-40      # below the floor: the block's codes are zero, its scale the floor's
    x[256:384] = 3e38 * torch.sign(rnd((128, 128), 3))
    x[384, 7], x[384, 8] = float("inf"), 1.0
    x[512, 9], x[512, 10] = float("nan"), 2.0
    q, scale = hc.quantize_fp8_block(x.cuda(), block_rows)
    back = hc.dequantize_fp8_block(q, scale, torch.float32, block_rows).cpu()
    scale = scale.cpu()
    assert torch.equal(back[:256], torch.zeros(256, 128))
    assert scale[0, 0] == torch.tensor(R.FLOOR) / 448
    assert bool(((back[256:384] - x[256:384]).abs() <= 3e38 * 2.0**-22).all())
    rows = slice(None) if block_rows == 128 else slice(0, 1)
    assert bool(back[384:512][rows].isnan().all()) and bool(back[512:][rows].isnan().all())
    if block_rows == 1:  # the other rows of the tile are blocks of their own
        assert torch.equal(back[385:512], torch.zeros(127, 128)) and torch.equal(back[513:], torch.zeros(127, 128))


@pytest.mark.parametrize("kind", KINDS)
def test_quantize_unaligned_buffers(cuda, kind):
    """A contiguous view that starts off a 16-byte boundary takes the same values."""
    x = rnd((1 + 6 * 256,), 4, kind).cuda()[1:].view(6, 256)
    q, scale = hc.quantize_fp8_block(x)
    ref_q, ref_s = R.quantize_rows(x.cpu())
    assert torch.equal(scale.cpu(), ref_s)
    same_codes(q, ref_q, "codes")
    qv = torch.empty(1 + 6 * 256, dtype=torch.uint8, device="cuda")[1:].view(6, 256)
    qv.copy_(q.view(torch.uint8))
    dy = rnd((6, 256), 5, kind).cuda()
    a = hc.activation_gelu_silu_ckpt_bwd(dy, qv.view(F8), scale, "gelu")
    assert torch.equal(a, hc.activation_gelu_silu_ckpt_bwd(dy, q, scale, "gelu"))


# ------------------------------------------------------------------------------ activation
@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", [(1, 1), (3, 127), (2, 128), (33, 1000), (5, 1001), (2, 3, 520), (257, 512)], ids=str)
def test_activation_ckpt(cuda, shape, kind, act):
    k = 0 if act == "gelu" else 1
    x = rnd(shape, 6, kind, 2.0)
    y, q, scale = hc.activation_gelu_silu_ckpt(x.cuda(), act)
    assert torch.equal(y, hc.activation_gelu_silu(x.cuda(), act))
    ref_q, ref_s = R.quantize_rows(x)
    assert torch.equal(scale.cpu(), ref_s)
    same_codes(q, ref_q, "codes")
    dy = rnd(shape, 7, kind)
    dx = hc.activation_gelu_silu_ckpt_bwd(dy.cuda(), q, scale, act)
    at = (ref_q * ref_s.repeat_interleave(128, -1)[..., : shape[-1]]).double()
    _, slope, _ = R.act(at, k)
    bound = dy.double().abs() * R.slope_bound(at, k) + 2 * R.U * (dy.double() * slope).abs()
    R.assert_within(dx, dy.double() * slope, bound, "dx")
    # along a direction: the difference of the 64-bit forward at the kept values
    v, h = rnd(shape, 8).double(), 1e-5
    diff = ((R.act(at + h * v, k)[0] - R.act(at - h * v, k)[0]) / (2 * h) * dy.double()).sum()
    slack = (bound + R.half_step(dx.dtype) * (dy.double() * slope).abs() + R.tiny(dx.dtype)) * v.abs()
    # central difference: h^2 / 6 of the third derivative (below 4 for both), and 2^-52 / h of the values
    slack = slack + dy.double().abs() * (h * h * v.abs() ** 3 * 4 + 1e-10 * (1 + at.abs()))
    assert abs(float((dx.cpu().double() * v).sum() - diff)) <= float(slack.sum())


@pytest.mark.parametrize("act,limit", [("gelu", 16.0), ("silu", 200.0)])
@pytest.mark.parametrize("kind", KINDS)
def test_activation_ckpt_far_values(cuda, kind, act, limit):
    """Slopes at large magnitudes are the limits 0 and 1, and a block with a NaN or an infinity gives NaN."""
    big = {"f32": 1e30, "bf16": 1e30, "f16": 6e4}[kind]
    x = torch.zeros(3, 256)
    x[0, :128] = torch.tensor([big, -big] * 64)
    x[0, 128:] = torch.tensor([limit * 1.5, -limit * 1.5] * 64)
    x[1, 0], x[2, 130] = float("nan"), float("inf")
    x = x.to(R.DTYPES[kind]).cuda()
    _, q, scale = hc.activation_gelu_silu_ckpt(x, act)
    dx = hc.activation_gelu_silu_ckpt_bwd(torch.ones_like(x), q, scale, act).float().cpu()
    expect = torch.tensor([1.0, 0.0] * 128)
    assert bool(((dx[0] - expect).abs() <= 2 * R.U).all())
    assert bool(dx[1, :128].isnan().all()) and bool((dx[1, 128:] == 0.5).all())
    assert bool(dx[2, 128:].isnan().all()) and bool((dx[2, :128] == 0.5).all())


@pytest.mark.parametrize("act", [0, 1])
def test_activation_autograd(ops, act):
    x = rnd((37, 264), 9, "bf16").cuda().requires_grad_(True)
    dy = rnd((37, 264), 10, "bf16").cuda()
    y, q, scale = ops.activation_gelu_silu_ckpt(x, act)
    assert y.requires_grad and not scale.requires_grad and not q.requires_grad
    (dx,) = torch.autograd.grad(y, x, dy)
    assert torch.equal(dx, ops.activation_gelu_silu_ckpt_bwd(dy, q, scale, act))
    y, _, _ = ops.activation_gelu_silu_ckpt(x, act)
    y.sum().backward()  # an expanded gradient
    assert torch.equal(x.grad, ops.activation_gelu_silu_ckpt_bwd(torch.ones_like(x), q, scale, act))
    y, _, _ = ops.activation_gelu_silu_ckpt(x, act)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(y, x, dy, create_graph=True)


# ------------------------------------------------------------------------------ matrix product
def operands(M, N, K, seed):
    a_q, a_s = hc.quantize_fp8_block(rnd((M, K), seed).cuda())
    w_q, w_s = hc.quantize_fp8_block((rnd((N, K), seed + 1) / math.sqrt(K)).cuda(), 128)
    return a_q, a_s, w_q, w_s


def check_product(c, a_q, a_s, w_q, w_s, bias):
    a, w = R.values(a_q, a_s), R.values(w_q, w_s, 128)
    ref, size = a @ w.t(), a.abs() @ w.abs().t()
    K = a.shape[1]
    # a block's 128 products are added, scaled and added to the blocks before: each addition off by
    # at most a whole step (a tensor core may truncate) of the magnitudes' sum; two scalings
    bound = 2 * R.U * (128 + -(-K // 128) + 6) * size
    if bias is not None:
        ref, bound = ref + bias.double(), bound + 2 * R.U * (size + bias.double().abs())
    R.assert_within(c, ref, bound, f"product {tuple(c.shape)} K {K}")


MNK = [(1, 1, 1), (1, 128, 128), (2, 7, 16), (3, 130, 48), (1, 512, 2048), (16, 256, 1040), (17, 384, 256), (33, 129, 144),
       (64, 1000, 512), (65, 257, 2064), (127, 640, 384), (128, 128, 4096), (129, 300, 272), (255, 1024, 640),
       (256, 256, 128), (300, 520, 1040), (513, 700, 896), (1024, 768, 1536), (2049, 2304, 272)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("M,N,K", MNK)
def test_matmul(cuda, M, N, K, kind):
    ops4 = operands(M, N, K, 11)
    for bias in (None, rnd((N,), 13, kind).cuda()):
        c = hc.matmul_fp8_block(*ops4, bias, R.DTYPES[kind])
        check_product(c, *ops4, bias)
    hc.check_device_error()


# (M, N, K, path): pairs with rows of C that are whole packs, whole words, and neither; several tiles per
# pair; one K block and fewer blocks than a group of scales; then the few-token kernel with its
# clusters of 1 to 8 CTAs and each of its token tiles
PATHS = [(2500, 2304, 400, 3), (2311, 2310, 1040, 3), (2305, 2561, 2064, 3), (4100, 4099, 128, 3), (5000, 2055, 1168, 3),
         (9000, 4000, 272, 3), (1, 6272, 2048, 1), (2, 3712, 2560, 1), (7, 3000, 3056, 1), (1, 2688, 3584, 1),
         (20, 384, 8192, 1), (48, 20000, 512, 1), (90, 777, 4096, 1), (96, 1030, 144, 1), (100, 4001, 1024, 1),
         (200, 257, 16384, 1)]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("M,N,K,path", PATHS)
def test_matmul_paths(cuda, M, N, K, path, kind):
    ops4 = operands(M, N, K, 12)
    bias = rnd((N,), 13, kind).cuda()
    c = hc.matmul_fp8_block(*ops4, bias, R.DTYPES[kind])
    assert hc.load().hc_matmul_fp8_block_last_path() == path
    check_product(c, *ops4, bias)
    hc.check_device_error()


def test_matmul_output_past_32_bits(cuda):
    """More than 2^32 elements of C: the last rows are those of the same product on its own."""
    M, N, K = 66000, 65600, 128
    a_q, a_s, w_q, w_s = operands(300, N, K, 28)
    big = a_q.view(torch.uint8).repeat(M // 300 + 1, 1)[:M].contiguous().view(F8)
    c = hc.matmul_fp8_block(big, a_s.repeat(M // 300 + 1, 1)[:M].contiguous(), w_q, w_s)
    first = M // 300 * 300
    assert torch.equal(c[first:], c[:M - first]) and torch.equal(c[first - 300:first], c[:300])
    check_product(c[M - 3:], big[M - 3:], a_s.repeat(M // 300 + 1, 1)[M - 3:M].contiguous(), w_q, w_s, None)


@pytest.mark.parametrize("M,N,K", [(5, 9, 33), (40, 130, 200), (300, 260, 1001), (1, 64, 8)])
def test_matmul_rows_of_any_length(cuda, M, N, K):
    """K that is no multiple of 16 runs on the SIMT kernel."""
    ops4 = operands(M, N, K, 14)
    check_product(hc.matmul_fp8_block(*ops4, None, torch.float32), *ops4, None)
    assert hc.load().hc_matmul_fp8_block_last_path() == 2


@pytest.mark.parametrize("M,N,K", [(3, 64, 128), (300, 300, 256)])
def test_matmul_unaligned_buffers(cuda, M, N, K):
    a_q, a_s, w_q, w_s = operands(M, N, K, 15)
    moved = torch.empty(1 + M * K, dtype=torch.uint8, device="cuda")[1:].view(M, K)
    moved.copy_(a_q.view(torch.uint8))
    check_product(hc.matmul_fp8_block(moved.view(F8), a_s, w_q, w_s), a_q, a_s, w_q, w_s, None)
    # scales and bias off a 16-byte boundary, outputs of every alignment that a row of C can have
    s1 = torch.empty(1 + a_s.numel(), device="cuda")[1:].view(a_s.shape).copy_(a_s)
    s2 = torch.empty(3 + w_s.numel(), device="cuda")[3:].view(w_s.shape).copy_(w_s)
    bias = torch.randn(N + 1, device="cuda")[1:].contiguous()
    check_product(hc.matmul_fp8_block(a_q, s1, w_q, s2, bias, torch.float32), a_q, a_s, w_q, w_s, bias)


def test_matmul_exact_small_integers(cuda):
    """Operands of small whole numbers with scales of powers of two: every product and sum is exact,
    so the result is too, whatever the order of additions."""
    g = torch.Generator().manual_seed(16)
    for M, N, K in ((1, 200, 512), (48, 272, 400), (300, 512, 1040)):
        a = torch.randint(-4, 5, (M, K), generator=g).float()
        w = torch.randint(-4, 5, (N, K), generator=g).float()
        a_s = 2.0 ** torch.randint(-2, 3, (M, -(-K // 128)), generator=g).float()
        w_s = 2.0 ** torch.randint(-2, 3, (-(-N // 128), -(-K // 128)), generator=g).float()
        dev = [a.to(F8).cuda(), a_s.cuda(), w.to(F8).cuda(), w_s.cuda()]
        ref = (R.values(dev[0], dev[1]) @ R.values(dev[2], dev[3], 128).t()).float()
        assert torch.equal(hc.matmul_fp8_block(*dev, None, torch.float32), ref), (M, N, K)


def test_matmul_nan_and_inf_stay_in_their_row(cuda):
    """A token whose block is NaN spoils its own output row only; an infinite weight scale its own 128 columns."""
    for M, N, K in ((4, 384, 256), (300, 384, 256)):
        a_q, a_s, w_q, w_s = operands(M, N, K, 17)
        a_s[2, 1] = float("nan")
        w_s[1, 0] = float("inf")
        c = hc.matmul_fp8_block(a_q, a_s, w_q, w_s, None, torch.float32)
        assert bool(c[2].isnan().all())
        rest = torch.cat([c[:2], c[3:]])
        assert bool((~rest[:, 128:256].isfinite()).all())
        assert bool(rest[:, :128].isfinite().all()) and bool(rest[:, 256:].isfinite().all())


def test_matmul_is_repeatable(cuda):
    for M, N, K in ((1, 4096, 4096), (200, 1024, 2048), (600, 1024, 1024)):
        ops4 = operands(M, N, K, 18)
        first = hc.matmul_fp8_block(*ops4)
        for _ in range(5):
            assert torch.equal(hc.matmul_fp8_block(*ops4), first)


def test_matmul_rows_do_not_depend_on_the_batch(cuda):
    """Each row of C is the same product whatever rows stand beside it, within the bound; rows behind
    the last one stay as they were."""
    M, N, K = 70, 256, 512
    a_q, a_s, w_q, w_s = operands(M, N, K, 19)
    buf = torch.full((M + 60, N), 7.0, dtype=torch.bfloat16, device="cuda")
    t = hc.MatmulFp8BlockTiling(M, K, N)
    for m in (M, 1, 33):
        buf.fill_(7.0)
        t.M = m
        hc.check(hc.load().hc_matmul_fp8_block_launch(a_q.data_ptr(), a_s.data_ptr(), w_q.data_ptr(), w_s.data_ptr(), None,
                                                      buf.data_ptr(), t, hc.DT_BF16,
                                                      torch.cuda.current_stream().cuda_stream))
        check_product(buf[:m], a_q[:m], a_s[:m], w_q, w_s, None)
        assert bool((buf[m:] == 7.0).all())


@pytest.mark.parametrize("cols", [128, 520])
def test_more_than_32_bits_of_elements(ops, cols):
    """Over 2^32 elements: the last rows of a tensor of repeated rows equal the first."""
    part = rnd((512, cols), 29, "bf16").cuda()
    n = (1 << 32) // (512 * cols) + 2
    x = part.repeat(n, 1)
    assert x.numel() > 1 << 32
    y, q, scale = ops.activation_gelu_silu_ckpt(x, 1)
    y0, q0, s0 = ops.activation_gelu_silu_ckpt(part, 1)
    for at in (0, n // 2, n - 1):
        rows = slice(512 * at, 512 * (at + 1))
        assert torch.equal(y[rows], y0) and torch.equal(scale[rows], s0)
        assert torch.equal(q[rows].view(torch.uint8), q0.view(torch.uint8))
    dx = ops.activation_gelu_silu_ckpt_bwd(x, q, scale, 1)
    assert torch.equal(dx[-512:], ops.activation_gelu_silu_ckpt_bwd(part, q0, s0, 1))


# ------------------------------------------------------------------------------ streams, graphs, together
def test_other_stream_and_empty_tensors(ops):
    s = torch.cuda.Stream()
    x = rnd((64, 512), 20, "bf16").cuda()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        q, scale = ops.quantize_fp8_block(x)
    s.synchronize()
    assert torch.equal(q.float().cpu(), R.quantize_rows(x.cpu())[0])
    for shape in ((0, 128), (3, 0), (2, 0, 5)):
        e = torch.empty(*shape, dtype=torch.bfloat16, device="cuda")
        q, scale = ops.quantize_fp8_block(e)
        assert q.shape == e.shape and scale.shape == (*shape[:-1], -(-shape[-1] // 128))
        y, q, scale = ops.activation_gelu_silu_ckpt(e, 0)
        assert ops.activation_gelu_silu_ckpt_bwd(y, q, scale, 0).shape == e.shape
    a = torch.empty(0, 128, device="cuda").to(F8)
    w_q, w_s = ops.quantize_fp8_block(rnd((64, 128), 21).cuda(), 128)
    assert ops.matmul_fp8_block(a, torch.empty(0, 1, device="cuda"), w_q, w_s, None, torch.bfloat16).shape == (0, 64)


def test_two_threads_on_two_streams(ops):
    """Both kinds of tensor-core kernel, the layer norm's gradients and the activation, called by two threads at
    once, each on its own stream: the bits of the calls alone."""
    import threading

    products = [operands(M, N, K, 30 + M) for M, N, K in ((16, 4096, 2048), (64, 2048, 4096), (100, 1024, 1024), (600, 1024, 1024))]
    x, dy = (rnd((300, 1024), s, "bf16").cuda() for s in (40, 41))
    gamma, beta = rnd((1024,), 42).cuda(), rnd((1024,), 43).cuda()

    def calls():
        out = [ops.matmul_fp8_block(*p, None, torch.bfloat16) for p in products]
        y, mean, rstd = ops.layer_norm_fwd_train(x, gamma, beta, 1e-5)
        out += [y, mean, rstd, *ops.layer_norm_bwd(dy, x, gamma, mean, rstd)]
        y, q, scale = ops.activation_gelu_silu_ckpt(x, 0)
        return out + [y, scale, ops.activation_gelu_silu_ckpt_bwd(dy, q, scale, 0)]

    want = calls()
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                got[i].append(calls())
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert [len(g) for g in got] == [10, 10]
    for g in got:
        for outs in g:
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_tensors_on_another_device(ops):
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    x = rnd((200, 512), 44, "bf16")
    gamma, beta = rnd((512,), 45), rnd((512,), 46)
    w = operands(200, 256, 512, 47)
    outs = []
    for d in (0, 1):
        on = [t.to(f"cuda:{d}") for t in (x, gamma, beta, *w)]
        with torch.cuda.device(0):  # the current device stays the first
            y, q, scale, rstd = ops.layer_norm_ckpt(*on[:3], 1e-5)
            grads = ops.layer_norm_ckpt_bwd(on[0], q, scale, on[1], rstd)
            outs.append([t.cpu() for t in (y, scale, rstd, *grads, ops.matmul_fp8_block(*on[3:], None, torch.float32),
                                           hc.matmul_fp8_block(*on[3:]))])
            assert torch.cuda.current_device() == 0
    assert all(torch.equal(a, b) for a, b in zip(*outs))


def feed_forward(ops, x, gamma, beta, w1, w2, dout):
    """One training step of a feed-forward layer with 8-bit operands and checkpoints: out, and the
    gradients of x, gamma, beta and both weights (bf16 [N, K])."""
    f8, bf = F8, torch.bfloat16

    def transposed(q, s):
        return ops.transpose_2d_4d(q.view(torch.uint8), 0).view(f8), s.t().contiguous()

    def linear(x, w):  # forward product; what its backward needs
        xq, w = ops.quantize_fp8_block(x), ops.quantize_fp8_block(w, 128)
        return ops.matmul_fp8_block(*xq, *w, None, bf), xq, w

    def linear_bwd(dy, xq, w):
        dx = ops.matmul_fp8_block(*ops.quantize_fp8_block(dy), *transposed(*w), None, bf)
        return dx, ops.matmul_bias(ops.transpose_2d_4d(dy, 0), ops.dequantize_fp8_block(*xq, bf))

    y, ln_q, ln_s, rstd = ops.layer_norm_ckpt(x, gamma, beta, 1e-5)
    h, yq, w1q = linear(y, w1)
    a, act_q, act_s = ops.activation_gelu_silu_ckpt(h, 0)
    out, aq, w2q = linear(a, w2)
    da, dw2 = linear_bwd(dout, aq, w2q)
    dh = ops.activation_gelu_silu_ckpt_bwd(da, act_q, act_s, 0)
    dy, dw1 = linear_bwd(dh, yq, w1q)
    dx, dgamma, dbeta = ops.layer_norm_ckpt_bwd(dy, ln_q, ln_s, gamma, rstd)
    return {"out": out, "dx": dx, "dgamma": dgamma, "dbeta": dbeta, "dw1": dw1, "dw2": dw2}


def feed_forward_inputs(rows, hidden, inner):
    x = rnd((rows, hidden), 22, "bf16").cuda()
    gamma, beta = 1 + 0.1 * rnd((hidden,), 23).cuda(), 0.1 * rnd((hidden,), 24).cuda()
    w1 = (rnd((inner, hidden), 25) / math.sqrt(hidden)).to(torch.bfloat16).cuda()
    w2 = (rnd((hidden, inner), 26) / math.sqrt(inner)).to(torch.bfloat16).cuda()
    return x, gamma, beta, w1, w2, rnd((rows, hidden), 27, "bf16").cuda()


@pytest.mark.parametrize("rows,hidden,inner", [(200, 256, 640), (512, 512, 1024), (8, 384, 128)])
def test_feed_forward_step(ops, rows, hidden, inner):
    """The step against the same step in 64 bits without any rounding.  Each rounding to e4m3 moves a
    tensor by at most 2^-4 of its norm (usually by 2^-5.3), each to bf16 by 2^-9; the longest chain
    (dx) passes ten tensors rounded to e4m3 (operands of four products, two checkpoints), so its
    norm may be off by up to (1 + 2^-4)^10 - 1 = 0.83, and by sqrt(10) 2^-5.3 = 0.08 where the roundings
    are independent: 0.2 leaves room for cancellation, while a wrong scale, transpose or block gives
    an error of the order of 1."""
    args = feed_forward_inputs(rows, hidden, inner)
    got = feed_forward(ops, *args)
    x, gamma, beta, w1, w2, dout = (t.double().requires_grad_(True) for t in args)
    y = R.layer_norm(x, gamma, beta, 1e-5)[0]
    out = R.act(y @ w1.t(), 0)[0] @ w2.t()
    grads = torch.autograd.grad(out, (x, gamma, beta, w1, w2), dout.detach())
    for name, ref in zip(("out", "dx", "dgamma", "dbeta", "dw1", "dw2"), (out, *grads)):
        err = float((got[name].double() - ref.detach()).norm() / ref.detach().norm())
        assert err <= 0.2, (name, err)
    hc.check_device_error()


def test_feed_forward_step_in_a_graph(ops):
    """Captured once, replayed on new inputs, two graphs in turn: the results are those of plain calls."""
    sets = [feed_forward_inputs(96, 256, 384), feed_forward_inputs(300, 256, 512)]
    graphs = []
    for args in sets:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            feed_forward(ops, *args)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = feed_forward(ops, *args)
        graphs.append((graph, out))
    for turn in range(3):
        for args, (graph, out) in zip(sets, graphs):
            args[0].copy_(rnd(tuple(args[0].shape), 30 + turn, "bf16"))
            graph.replay()
            plain = feed_forward(ops, *args)
            for name in plain:
                assert torch.equal(plain[name], out[name]), (turn, name)
