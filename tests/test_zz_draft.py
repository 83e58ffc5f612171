import math
import numpy as np
import pytest
import torch
from test_gqa_gpu import *
from test_gqa_gpu import check_decode, check_weights, Cache, rand, status, U, G, f64
pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- A
def pool(nb, page, hkv, d, seed):
    """A filled cache: k_cache, v_cache, k_scale, v_scale."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = [(torch.randn(nb, page, hkv, d, generator=g, device="cuda") * 60).clamp_(-448, 448).to(torch.float8_e4m3fn)
         for _ in range(2)]
    return x + [torch.exp2(torch.randint(-8, -4, (nb, hkv), generator=g, device="cuda").float()) for _ in range(2)]


def check_decode_on_gpu(dev, q, scale=None):
    """check_decode for long contexts, with the 64-bit sums on the GPU.  A
    weight's rounding to fp16 is off by no more than the weight itself, and
    a warp's sums have four steps for each of its units, each off by 2^-23 at
    most."""
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
            e = 2.0 ** -19 * size + 2.0 ** -20 + steps
            tol = u * want.abs() + (2.0 ** -11 + 2 * e)[..., None] * mag + rest + 1e-30
            o, l = got[i, :, kvh * g:(kvh + 1) * g].double(), lse[i, kvh * g:(kvh + 1) * g].T.double()
            off = (o - want).abs()
            assert (off <= tol).all(), (i, kvh, off.max().item(), tol[off > tol].min().item() if (off > tol).any() else "not finite", int((~(off <= tol)).sum()))
            none = ~sees.any(-1)
            assert torch.isneginf(l[none]).all()
            assert ((l - wl).abs() <= e + 2.0 ** -22 * wl.abs())[~none].all(), (i, kvh)
    return got, lse


Z = "zero"
SCALES = {"zero blocks": [17, Z, -8, 17, Z], "large": [119, -8, 119, Z, 3], "upwards": [-8, 60, 119],
          "downwards": [100, 50, 0, -50, -100, -126], "tiny": [0, -127, -140, -8], "near": [-8, -30, -7, -50]}


@pytest.mark.parametrize("h,d,page", [(4, 128, 16), (16, 128, 64), (3, 64, 32), (12, 64, 16)])
@pytest.mark.parametrize("kind", SCALES)
def test_decode_value_scales_far_apart(kind, h, d, page):
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
    check_decode_on_gpu((kc, vc, ks, vs, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")), rand(g, len(lens), 1, h, d))


def test_decode_after_append_of_zeros():
    import deepseek_v4_kernel as dk
    kc, vc, ks, vs = pool(4, 16, 1, 128, 42)
    table, ctx = torch.arange(4, dtype=torch.int32, device="cuda")[None], torch.tensor([48], dtype=torch.int32, device="cuda")
    k, v = torch.zeros(48, 1, 128, dtype=torch.bfloat16, device="cuda"), torch.zeros(48, 1, 128, dtype=torch.bfloat16, device="cuda")
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
    dev = (kc, vc, ks, vs, torch.arange(64, dtype=torch.int32, device="cuda")[None], torch.tensor([1020], dtype=torch.int32, device="cuda"))
    check_decode_on_gpu(dev, torch.full((1, 1, 3, 128), -16.0, dtype=torch.bfloat16, device="cuda"))


# ---------------------------------------------------------------- B
@pytest.mark.parametrize("top", [116, 120, 127])
def test_queries_near_the_largest(top):
    g = torch.Generator(device="cuda").manual_seed(44)
    c = Cache([300, 64], 16, 2, 128, seed=12)
    c.ks *= 2.0 ** (-top)
    def big(s_q):
        q = (torch.randn(2, s_q, 8, 128, generator=g, device="cuda") * 0.25).clamp(-0.99, 0.99)
        return (q.double() * 2.0 ** top).bfloat16()
    q = big(1)
    assert q.isfinite().all()
    check_decode(c, q)
    check_weights(c, q)
    check_weights(c, big(10))


# ---------------------------------------------------------------- C
@pytest.mark.parametrize("s_q", [1, 3, 40, 60])
@pytest.mark.parametrize("what", [float("nan"), float("inf")])
def test_weights_of_queries_that_are_left_out(s_q, what):
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


# ---------------------------------------------------------------- D
LONG = [(4, 1, 1, 128, 256, [130001, 0, 70, 1, 64, 33000, 8193, 60000]), (16, 2, 1, 64, 16, [65, 50000, 0, 128, 12345, 70007]),
        (1, 1, 2, 64, 64, [300000, 3, 100000, 1]), (24, 2, 3, 128, 64, [20011, 5, 0, 40000, 64]), (32, 8, 1, 128, 32, [9000 + 77 * i for i in range(24)]),
        (40, 8, 2, 64, 128, [1 + 531 * i for i in range(40)])]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("h,hkv,sq,d,page,lens", LONG)
@pytest.mark.parametrize("grow", [False, True])
def test_decode_many_units_of_every_warp(h, hkv, sq, d, page, lens, grow, dtype):
    g = torch.Generator(device="cuda").manual_seed(46)
    nb = 700
    kc, vc, ks, vs = pool(nb, page, hkv, d, 47)
    width = max(-(-n // page) for n in lens)
    table = torch.randint(nb, (len(lens), width), generator=g, device="cuda", dtype=torch.int32)
    if grow:  # scores that grow along the context
        table = table.sort(1)[0]
        ks *= torch.exp2(torch.linspace(-4, 3, nb, device="cuda"))[:, None]
    q = rand(g, len(lens), sq, h, d, dtype=dtype)
    check_decode_on_gpu((kc, vc, ks, vs, table, torch.tensor(lens, dtype=torch.int32, device="cuda")), q)


# ---------------------------------------------------------------- E
def test_decode_long_tail_of_small_weights():
    """2^14 weights of 2^-26.5 of the largest, whose value is zero: they make the output."""
    import deepseek_v4_kernel as dk
    n, b = 1 << 14, 12 * torch.cuda.get_device_properties(0).multi_processor_count
    kc, vc = (torch.zeros(16, 1024, 1, 64, dtype=torch.uint8, device="cuda") for _ in range(2))
    kc[0, 0], vc[:] = 0x38, 0x38
    vc[0, 0] = 0
    one = torch.ones(16, 1, device="cuda")
    table = torch.arange(16, dtype=torch.int32, device="cuda").expand(b, 16).contiguous()
    ctx = torch.full((b,), n, dtype=torch.int32, device="cuda")
    q = torch.ones(b, 1, 1, 64, dtype=torch.bfloat16, device="cuda")
    out, lse = dk.gqa_decode_fwd(q, kc, vc, one, one, table, ctx, sm_scale=26.5 * math.log(2) / 64)
    tail = (n - 1) * 2.0 ** -26.5
    want = tail / (1 + tail)
    off = (out.double() - want).abs().max().item()
    assert off <= 2.0 ** -8 * want + n * 2.0 ** -32, (off, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prefill_long_tail_of_small_weights(dtype):
    import deepseek_v4_kernel as dk
    n = 1 << 14
    q = torch.ones(1, 1, 64, dtype=dtype, device="cuda")
    k, v = torch.zeros(n, 1, 64, dtype=dtype, device="cuda"), torch.ones(n, 1, 64, dtype=dtype, device="cuda")
    k[0], v[0] = 1, 0
    cq, ck = (torch.tensor([0, x], dtype=torch.int32, device="cuda") for x in (1, n))
    out, lse = dk.gqa_prefill_fwd(q, k, v, cq, ck, sm_scale=26.5 * math.log(2) / 64)
    tail = (n - 1) * 2.0 ** -26.5
    want = tail / (1 + tail)
    off = (out.double() - want).abs().max().item()
    assert off <= 2 * U[dtype] * want + n * 2.0 ** -32, (off, want)


# ---------------------------------------------------------------- F
def test_status_of_a_device_without_an_index():
    import deepseek_v4_kernel as dk
    assert dk.gqa_status(torch.device("cuda")) == 0


def test_out_may_be_q():
    import deepseek_v4_kernel as dk
    g = torch.Generator(device="cuda").manual_seed(48)
    c = Cache([3000, 40, 900], 64, 2, 128, seed=14)
    dev, q = c.cuda(), rand(g, 3, 5, 8, 128)
    o, l = dk.gqa_decode_fwd(q, *dev)
    x, kv = rand(g, 1500, 8, 128), rand(g, 1500, 2, 128)
    cu = torch.tensor([0, 900, 1000, 1500], dtype=torch.int32, device="cuda")
    po, pl = dk.gqa_prefill_fwd(x, kv, kv, cu)
    o2, l2 = dk.gqa_decode_fwd(q, *dev, out=q)
    po2, pl2 = dk.gqa_prefill_fwd(x, kv, kv, cu, out=x)
    assert torch.equal(o, o2) and torch.equal(l, l2) and torch.equal(po, po2) and torch.equal(pl, pl2)


def test_repeats_bit_for_bit_long():
    import deepseek_v4_kernel as dk
    g = torch.Generator(device="cuda").manual_seed(49)
    x, kv = rand(g, 6000, 8, 128), rand(g, 6000, 2, 128)
    cu = torch.tensor([0, 4099, 5000, 6000], dtype=torch.int32, device="cuda")
    kc, vc, ks, vs = pool(700, 64, 2, 128, 47)
    table = torch.randint(700, (4, 1000), generator=g, device="cuda", dtype=torch.int32)
    ctx = torch.tensor([64000, 1, 33333, 50], dtype=torch.int32, device="cuda")
    q = rand(g, 4, 1, 8, 128)
    def run():
        o, l = dk.gqa_decode_fwd(q, kc, vc, ks, vs, table, ctx)
        return dk.gqa_prefill_fwd(x, kv, kv, cu) + (o, l, dk.gqa_attention_weights(q, l, kc, ks, table, ctx))
    first = run()
    for _ in range(20):
        for a, b in zip(first, run()):
            assert torch.equal(a, b)
