"""Grouped-query operators on the GPU at the ends of their range: magnitudes
and scales far apart, contexts that give every warp many units, rows that are
left out, tensors that share memory.  Tolerances as in test_gqa_gpu.py, where
nothing else is said."""
import math

import pytest
import torch

from test_gqa_gpu import Cache, U, check_decode, check_weights, rand, status

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ prompts
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prefill_long_tail_of_small_weights(dtype):
    """As test_decode_long_tail_of_small_weights, of one query over a long
    context; P is rounded to the inputs' type."""
    import deepseek_v4_kernel as dk
    n = 1 << 14
    q = torch.ones(1, 1, 64, dtype=dtype, device="cuda")
    k, v = torch.zeros(n, 1, 64, dtype=dtype, device="cuda"), torch.ones(n, 1, 64, dtype=dtype, device="cuda")
    k[0], v[0] = 1, 0
    cq, ck = (torch.tensor([0, x], dtype=torch.int32, device="cuda") for x in (1, n))
    out, lse = dk.gqa_prefill_fwd(q, k, v, cq, ck, sm_scale=26.5 * math.log(2) / 64)
    tail = (n - 1) * 2.0 ** -26.5
    want = tail / (1 + tail)
    assert (out.double() - want).abs().max() <= 2 * U[dtype] * want + n * 2.0 ** -32
    size = 26.5 * math.log(2)  # T, and nearly the lse: 2^-19 T + 2^-20 + 2^-22 |lse|
    assert abs(lse.item() - size - math.log1p(tail)) <= (2.0 ** -19 + 2.0 ** -22) * size + 2.0 ** -20
    assert status() == 0


# ------------------------------------------------------------------ decode
def pool(nb, page, hkv, d, seed):
    """A filled cache: k_cache, v_cache, k_scale, v_scale."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = [(torch.randn(nb, page, hkv, d, generator=g, device="cuda") * 60).clamp_(-448, 448).to(torch.float8_e4m3fn)
         for _ in range(2)]
    return x + [torch.exp2(torch.randint(-8, -4, (nb, hkv), generator=g, device="cuda").float()) for _ in range(2)]


def check_decode_on_gpu(dev, q, scale=None):
    """check_decode for long contexts, with the 64-bit sums on the GPU.  A
    weight's rounding to fp16 is off by no more than the weight itself, and
    a warp's sums have four steps for each of its units, off by 2^-23 each.  The
    sums are fp32 in units of up to the sequence's largest v_scale S, whether a
    row sees it or not: a smaller scale's factor is off by 2^-150, that times 448
    S, and 2^16 sums by steps of 2^-149 S over 2^7: 2^-139 S."""
    import deepseek_v4_kernel as dk
    kc, vc, ks, vs, table, ctx = dev
    b, s_q, h, d = q.shape
    page, hkv = kc.shape[1:3]
    g = h // hkv
    scale = d ** -0.5 if scale is None else scale
    got, lse = dk.gqa_decode_fwd(q, *dev, sm_scale=scale)
    torch.cuda.synchronize()
    assert status() == 0
    lens = ctx.tolist()
    units = sum(max(1, -(-n // 64)) for n in lens) * hkv * -(-g * s_q // 16)
    pieces = torch.cuda.get_device_properties(0).multi_processor_count * 8
    steps = 2.0 ** -23 * (4 * -(-units // pieces) + 32)
    u = U[q.dtype]
    least = 2.0 ** -25 if q.dtype == torch.float16 else 1e-30  # fp16 has steps of 2^-24 at zero
    for i, n in enumerate(lens):
        if n == 0:
            assert (got[i] == 0).all() and torch.isneginf(lse[i]).all()
            continue
        t = torch.arange(n, device="cuda")
        blk = table[i, t // page].long()
        sees = t <= n - s_q + torch.arange(s_q, device="cuda")[:, None]
        for kvh in range(hkv):
            k, v = (x[blk, t % page, kvh].double() * y[blk, kvh].double()[:, None] for x, y in ((kc, ks), (vc, vs)))
            rows = q[i, :, kvh * g:(kvh + 1) * g].double()
            s = torch.where(sees[:, None], rows @ k.T * scale, -math.inf)
            size = torch.where(sees[:, None], rows.abs() @ k.abs().T * scale, 0).amax(-1)
            wl = torch.logsumexp(s, -1)
            p = torch.where(sees[:, None], torch.exp(s - wl[..., None]), 0)
            want, mag, rest = p @ v, p @ v.abs(), p.clamp(max=2.0 ** -25) @ v.abs()
            most = vs[blk, kvh].double().max()
            e = 2.0 ** -19 * size + 2.0 ** -20 + steps
            err = (2.0 ** -11 + 2 * e)[..., None] * mag + rest + 2.0 ** -139 * most
            tol = u * (want.abs() + err) + err + least  # (what is rounded is off already)
            o, l = got[i, :, kvh * g:(kvh + 1) * g].double(), lse[i, kvh * g:(kvh + 1) * g].T.double()
            off = (o - want).abs()
            assert (off <= tol).all(), (i, kvh, off.max().item(), int((~(off <= tol)).sum()))
            none = ~sees.any(-1)
            assert torch.isneginf(l[none]).all()
            assert ((l - wl).abs() <= e + 2.0 ** -22 * wl.abs())[~none].all(), (i, kvh)
    return got, lse


Z = "zero"
SCALES = {"zero blocks": [17, Z, -8, 17, Z], "large": [119, -8, 119, Z, 3], "upwards": [-8, 60, 119],
          "downwards": [100, 50, 0, -50, -100, -126], "tiny": [0, -127, -140, -8], "near": [-8, -30, -7, -50]}


@pytest.mark.parametrize("h,d,page,s_q", [(4, 128, 16, 1), (16, 128, 64, 1), (3, 64, 32, 1), (12, 64, 16, 1), (2, 128, 16, 4),
                                          (5, 64, 16, 5), (1, 128, 32, 70)])
@pytest.mark.parametrize("kind", SCALES)
def test_decode_value_scales_far_apart(kind, h, d, page, s_q):
    """Blocks whose v_scale differ by up to 2^219, subnormal ones and blocks of zeros (Z) among them."""
    g = torch.Generator(device="cuda").manual_seed(40)
    lens = [(211 * i) % 1900 for i in range(120)] + [9000]
    counts = [-(-n // page) for n in lens]
    kc, vc, ks, vs = pool(sum(counts), page, 1, d, 41)
    table = torch.zeros(len(lens), max(counts), dtype=torch.int32)
    at = 0
    exps = torch.zeros(sum(counts), dtype=torch.float64)
    zero = torch.zeros(sum(counts), dtype=torch.bool)
    for i, c in enumerate(counts):
        table[i, :c] = torch.arange(at, at + c)
        for j in range(c):
            x = SCALES[kind][(i + j) % len(SCALES[kind])]
            zero[at + j] = x == Z
            exps[at + j] = -100 if x == Z else x
        at += c
    vs[:, 0] = torch.exp2(exps).float().cuda()
    vc.view(torch.uint8)[zero.cuda()] = 0
    ctx = torch.tensor(lens, dtype=torch.int32, device="cuda")
    check_decode_on_gpu((kc, vc, ks, vs, table.cuda(), ctx), rand(g, len(lens), s_q, h, d))


@pytest.mark.parametrize("exps", [[-8, Z, 119, -8], [-44, Z, 57, Z], [0, -60, 119, Z], [-30, Z, 119, 119]])
@pytest.mark.parametrize("h,d", [(3, 128), (12, 64)])
def test_decode_zeros_before_large_values_out_of_sight(exps, h, d):
    """The largest blocks have weights of 2^-261; zeros or small values stand
    between them and those that make the output."""
    lens = [64, 50, 700] * 40
    kc, vc, ks, vs = pool(44 * len(lens), 16, 1, d, 44)
    kc.zero_()
    ks.fill_(1.0)
    where = torch.arange(44 * len(lens), device="cuda") % 4
    top = max(x for x in exps if x != Z)
    for i, x in enumerate(exps):
        vs[where == i] = 2.0 ** (-100 if x == Z else x)
        if x == Z:
            vc.view(torch.uint8)[where == i] = 0
        elif x == top:
            kc.view(torch.uint8)[where == i] = 0x38  # 1.0
    table = torch.arange(44 * len(lens), dtype=torch.int32, device="cuda").view(len(lens), 44)
    q = torch.full((len(lens), 1, h, d), -16.0 * 128 / d, dtype=torch.bfloat16, device="cuda")
    check_decode_on_gpu((kc, vc, ks, vs, table, torch.tensor(lens, dtype=torch.int32, device="cuda")), q, scale=128 ** -0.5)


@pytest.mark.parametrize("exps", [[-80, 40], [118, -8], [-8, -8, 118, 60], [0, 100, -30]])
@pytest.mark.parametrize("h,d", [(2, 128), (8, 64)])
def test_decode_drafts_that_do_not_see_the_largest_values(exps, h, d):
    """Blocks of 16 whose v_scale lie up to 2^130 apart, queries that see one, two and more of them."""
    lens = list(range(1, 131))
    kc, vc, ks, vs = pool(9 * len(lens), 16, 1, d, 43)
    table = torch.arange(9 * len(lens), dtype=torch.int32, device="cuda").view(len(lens), 9)
    vs.view(len(lens), 9)[:] = torch.exp2(torch.tensor([exps[i % len(exps)] for i in range(9)]).float())
    ctx = torch.tensor(lens, dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(51)
    check_decode_on_gpu((kc, vc, ks, vs, table, ctx), rand(g, len(lens), 64, h, d))


def test_decode_after_append_of_zeros():
    """A block of zeros, which append gives the scale 2^-100, behind large values."""
    import deepseek_v4_kernel as dk
    kc, vc, ks, vs = pool(4, 16, 1, 128, 42)
    table = torch.arange(4, dtype=torch.int32, device="cuda")[None]
    ctx = torch.tensor([48], dtype=torch.int32, device="cuda")
    k, v = (torch.zeros(48, 1, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    v[:16] = 3e7
    v[32:] = 1.0
    cu = torch.tensor([0, 48], dtype=torch.int32, device="cuda")
    dk.gqa_cache_append(k, v, cu, ctx, table, kc, vc, ks, vs)
    check_decode_on_gpu((kc, vc, ks, vs, table, ctx), torch.zeros(1, 1, 2, 128, dtype=torch.bfloat16, device="cuda"))


@pytest.mark.parametrize("first", [True, False])
def test_decode_large_values_out_of_sight(first):
    """V of 2^119 units at positions of weight 2^-261, ordinary ones elsewhere."""
    kc, vc, ks, vs = pool(64, 16, 1, 128, 43)
    ks.fill_(1.0)
    kc.zero_()
    far = torch.zeros(64, dtype=torch.bool)
    far[0 if first else 9] = far[20:23] = True
    far = far.cuda()
    kc.view(torch.uint8)[far] = 0x38  # 1.0
    vs[far], vs[~far] = 2.0 ** 119, 2.0 ** -8
    table = torch.arange(64, dtype=torch.int32, device="cuda")[None]
    ctx = torch.tensor([1020], dtype=torch.int32, device="cuda")
    check_decode_on_gpu((kc, vc, ks, vs, table, ctx), torch.full((1, 1, 3, 128), -16.0, dtype=torch.bfloat16, device="cuda"))


@pytest.mark.parametrize("top", [116, 120, 127])
def test_queries_near_the_largest(top):
    """bf16 queries of up to 2^top beside keys as small: ordinary scores, in
    decode and in both kernels of the weights."""
    g = torch.Generator(device="cuda").manual_seed(44)
    c = Cache([300, 64], 16, 2, 128, seed=12)
    c.ks *= 2.0 ** -top
    for s_q in (1, 10):
        x = (torch.randn(2, s_q, 8, 128, generator=g, device="cuda") * 0.25).clamp(-0.99, 0.99)
        q = (x.double() * 2.0 ** top).bfloat16()
        assert q.isfinite().all()
        check_decode(c, q)
        check_weights(c, q)


LONG = [(4, 1, 1, 128, 256, [130001, 0, 70, 1, 64, 33000, 8193, 60000]),
        (16, 2, 1, 64, 16, [65, 50000, 0, 128, 12345, 70007]),
        (1, 1, 2, 64, 64, [300000, 3, 100000, 1]),
        (24, 2, 3, 128, 64, [20011, 5, 0, 40000, 64]),
        (16, 1, 1, 128, 16, [400000, 31, 250000]),
        (12, 1, 1, 64, 64, [1000003, 77, 0, 500000]),
        (32, 8, 1, 128, 32, [9000 + 77 * i for i in range(24)]),
        (64, 8, 1, 128, 64, [20000 + 3001 * i for i in range(20)]),
        (40, 8, 2, 64, 128, [1 + 531 * i for i in range(40)])]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("h,hkv,sq,d,page,lens", LONG)
@pytest.mark.parametrize("grow", [False, True])
def test_decode_many_units_of_every_warp(h, hkv, sq, d, page, lens, grow, dtype):
    """Rings that wrap, running maxima and sums carried from unit to unit, one
    (sequence, head, group) after another in a warp, pieces joined over warps
    and CTAs: 2 to 68 units of a warp, scales that differ from block to block."""
    g = torch.Generator(device="cuda").manual_seed(46)
    nb = 700
    kc, vc, ks, vs = pool(nb, page, hkv, d, 47)
    width = max(-(-n // page) for n in lens)
    table = torch.randint(nb, (len(lens), width), generator=g, device="cuda", dtype=torch.int32)
    if grow:  # scores that grow along the context
        table = table.sort(1)[0]
        ks *= torch.exp2(torch.linspace(-4, 3, nb, device="cuda"))[:, None]
    q = rand(g, len(lens), sq, h, d, dtype=dtype)
    ctx = torch.tensor(lens, dtype=torch.int32, device="cuda")
    check_decode_on_gpu((kc, vc, ks, vs, table, ctx), q)


def test_decode_long_tail_of_small_weights():
    """2^14 weights of 2^-26.5 of the largest, whose own value is zero, make the
    output.  In fp16 the largest weight is 2^7 at least, so that each of them is
    off by 2^-25 of that at most; a warp has a whole context."""
    import deepseek_v4_kernel as dk
    n, b = 1 << 14, 12 * torch.cuda.get_device_properties(0).multi_processor_count
    kc, vc = (torch.zeros(16, 1024, 1, 64, dtype=torch.uint8, device="cuda") for _ in range(2))
    kc[0, 0], vc[:] = 0x38, 0x38  # 1.0
    vc[0, 0] = 0
    one = torch.ones(16, 1, device="cuda")
    table = torch.arange(16, dtype=torch.int32, device="cuda").expand(b, 16).contiguous()
    ctx = torch.full((b,), n, dtype=torch.int32, device="cuda")
    q = torch.ones(b, 1, 1, 64, dtype=torch.bfloat16, device="cuda")
    out, _ = dk.gqa_decode_fwd(q, kc, vc, one, one, table, ctx, sm_scale=26.5 * math.log(2) / 64)
    tail = (n - 1) * 2.0 ** -26.5
    want = tail / (1 + tail)
    assert (out.double() - want).abs().max() <= U[q.dtype] * want + n * 2.0 ** -32
    assert status() == 0


# ------------------------------------------------------------------ weights
@pytest.mark.parametrize("s_q", [1, 3, 40, 60])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), 1.0])
def test_weights_of_queries_that_are_left_out(s_q, what):
    """An lse of -inf: the query adds nothing, whatever it holds; nor do
    positions that hold NaN where no query is left."""
    import deepseek_v4_kernel as dk
    g = torch.Generator(device="cuda").manual_seed(45)
    c = Cache([300, 128, 90], 32, 2, 128, seed=13)
    q = rand(g, 3, s_q, 4, 128)
    _, lse = dk.gqa_decode_fwd(q, *c.cuda())
    lse[0, 1, s_q // 2] = -math.inf
    q[0, s_q // 2, 1, 5:7] = what
    q[0, s_q // 2, 1, 9] = -what
    lse[2] = -math.inf
    q[2] = what
    c.kc[c.table[2, 0].item(), 3, :, 0] = 0x7F
    w = check_weights(c, q, lse=lse)
    assert (w[2] == 0).all()


# ------------------------------------------------------------------ arguments
@pytest.mark.parametrize("device", [None, "cuda", "cuda:0"])
def test_status_takes_any_form_of_a_device(device):
    import deepseek_v4_kernel as dk
    assert dk.gqa_status(device) == 0
    assert dk.gqa_status(None if device is None else torch.device(device)) == 0


def test_evict_weights_and_new_weights_of_one_tensor():
    """Column ranges of one tensor are taken, ranges that share an element are
    refused before anything is written."""
    import deepseek_v4_kernel as dk
    c = Cache([300, 150], 32, 2, 64, seed=15, spare=8)
    g = torch.Generator(device="cuda").manual_seed(50)
    w = torch.rand(2, 2, 300, generator=g, device="cuda")
    new = c.free[:8].int().view(2, 4).cuda()
    want = dk.gqa_cache_evict(*c.cuda(), w, 100, 10, new)
    both = torch.full((2, 2, 420), 3.0, device="cuda")
    both[..., :300] = w
    for into in (both[..., 300:410], both.transpose(0, 1)[..., 300:410]):
        got = dk.gqa_cache_evict(*c.cuda(), both[..., :300], 100, 10, new, new_weights=into)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1][..., :100], want[1]) and torch.equal(got[2], want[2])
        assert (both[..., 400:410] == 0).all() and (both[..., 410:] == 3.0).all() and torch.equal(both[..., :300], w)
    dev = c.cuda()
    before = [t.clone() for t in dev]
    for bad in (both[..., 4:104], both[..., 299:410], both[:, 1:].expand(2, 2, 420)):
        with pytest.raises(RuntimeError):
            dk.gqa_cache_evict(*dev, both[..., :300], 100, 10, new, new_weights=bad)
    torch.cuda.synchronize()
    assert all(torch.equal(t.view(torch.uint8), x.view(torch.uint8)) for t, x in zip(dev, before)) and status() == 0


def test_written_tensors_whose_rows_overlap_are_refused():
    import deepseek_v4_kernel as dk
    c = Cache([70, 64], 32, 2, 128, seed=1)
    kc, vc, ks, vs, table, ctx = dev = c.cuda()
    q = torch.zeros(2, 2, 4, 128, dtype=torch.bfloat16, device="cuda")
    lse = torch.zeros(2, 4, 2, device="cuda")
    half = torch.zeros(4096, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="overlap"):
        dk.gqa_decode_fwd(q, *dev, out=half.as_strided(q.shape, (512, 512, 128, 1)))
    with pytest.raises(RuntimeError, match="overlap"):
        dk.gqa_attention_weights(q, lse, kc, ks, table, ctx, weights=torch.zeros(500, device="cuda").as_strided((2, 2, 96), (96, 96, 1)))
    x = torch.zeros(9, 4, 128, dtype=torch.bfloat16, device="cuda")
    cu = torch.tensor([0, 9], dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="overlap"):
        dk.gqa_prefill_fwd(x, x, x, cu, out=half.as_strided(x.shape, (128, 128, 1)))


def test_arguments_past_their_types_are_refused():
    """Numbers that fp32 or 32 bits do not hold, tensors without dims: RuntimeError, before any memory is asked for."""
    import deepseek_v4_kernel as dk
    c = Cache([70, 64], 32, 2, 128, seed=1, spare=8)
    kc, vc, ks, vs, table, ctx = dev = c.cuda()
    q = torch.zeros(2, 1, 4, 128, dtype=torch.bfloat16, device="cuda")
    lse, w = torch.zeros(2, 4, 1, device="cuda"), torch.zeros(2, 2, 96, device="cuda")
    cu, new = torch.tensor([0, 1, 3], dtype=torch.int32, device="cuda"), c.free[:4].int().view(2, 2).cuda()
    x = torch.zeros(9, 4, 128, dtype=torch.bfloat16, device="cuda")
    cx = torch.tensor([0, 9], dtype=torch.int32, device="cuda")
    for scale in (3.5e38, 1e300, 1e-46):
        with pytest.raises(RuntimeError):
            dk.gqa_decode_fwd(q, *dev, sm_scale=scale)
        with pytest.raises(RuntimeError):
            dk.gqa_attention_weights(q, lse, kc, ks, table, ctx, sm_scale=scale)
        with pytest.raises(RuntimeError):
            dk.gqa_prefill_fwd(x, x, x, cx, sm_scale=scale)
    for width in ((1 << 30) + 1, (1 << 32) + 96, -(1 << 32) + 96):
        with pytest.raises(RuntimeError, match="max_context"):
            dk.gqa_attention_weights(q, lse, kc, ks, table, ctx, max_context=width)
        with pytest.raises(RuntimeError, match="budget"):
            dk.gqa_cache_evict(*dev, w, width, 4, new)
    wide = torch.zeros(1, device="cuda").expand(2, 2, (1 << 32) + 96)
    with pytest.raises(RuntimeError):
        dk.gqa_attention_weights(q, lse, kc, ks, table, ctx, weights=wide)
    for bad in (q[0, 0, 0, 0], q[0, 0, 0]):
        with pytest.raises(RuntimeError):
            dk.gqa_cache_append(bad, bad, cu, ctx, table, kc, vc, ks, vs)
    assert status() == 0


# ------------------------------------------------------------------ together
def test_out_may_be_q():
    import deepseek_v4_kernel as dk
    g = torch.Generator(device="cuda").manual_seed(48)
    c = Cache([3000, 40, 900], 64, 2, 128, seed=14)
    dev, q = c.cuda(), rand(g, 3, 5, 8, 128)
    x, kv = rand(g, 1500, 8, 128), rand(g, 1500, 2, 128)
    cu = torch.tensor([0, 900, 1000, 1500], dtype=torch.int32, device="cuda")
    want = dk.gqa_decode_fwd(q, *dev) + dk.gqa_prefill_fwd(x, kv, kv, cu)
    got = dk.gqa_decode_fwd(q, *dev, out=q) + dk.gqa_prefill_fwd(x, kv, kv, cu, out=x)
    assert got[0].data_ptr() == q.data_ptr() and got[2].data_ptr() == x.data_ptr()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and status() == 0


@pytest.mark.parametrize("s", [1, 24])
def test_weights_of_a_prompts_last_queries(s):
    """A prompt, its append, and the weights that its last queries gave the
    cached positions, with the prompt's own lse."""
    import deepseek_v4_kernel as dk
    g = torch.Generator(device="cuda").manual_seed(52)
    lens, h, hkv, d, page = [300, 24, 131], 8, 2, 128, 32
    cu = torch.tensor([0, 300, 324, 455], dtype=torch.int32, device="cuda")
    q, k, v = rand(g, 455, h, d), rand(g, 455, hkv, d), rand(g, 455, hkv, d)
    _, lse = dk.gqa_prefill_fwd(q, k, v, cu)
    c = Cache([0, 0, 0], page, hkv, d, seed=1, spare=30, width=10)
    c.table[:] = c.free[:30].view(3, 10)
    c.ctx = torch.tensor(lens, dtype=torch.int32)
    kc, vc, ks, vs, table, ctx = c.cuda()
    dk.gqa_cache_append(k, v, cu, ctx, table, kc, vc, ks, vs)
    c.kc, c.ks = kc.view(torch.uint8).cpu(), ks.cpu()
    rows = cu[1:, None].long() - s + torch.arange(s, device="cuda")
    check_weights(c, q[rows], lse=lse[rows].transpose(1, 2).contiguous())
