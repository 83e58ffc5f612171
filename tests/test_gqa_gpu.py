"""Grouped-query operators on the GPU against the float64 oracle
(oracle/gqa_oracle.py): packed prompts, and the e4m3 cache's append, decode,
attention weights and eviction.

Tolerances, from the roundings that each kernel makes (u = half a step of
the type, relative to the value: bf16 2^-8, fp16 2^-11):

* a score's fp32 sum over d, in at most 12 accumulating steps that may each
  truncate: ds <= 16 * 2^-23 T, T the largest sm_scale * sum |q||k| of the
  row; scaling it, subtracting the maximum and exp2 (2 ulp) add less than
  2^-21 (1 + T): a weight p is off by e = 2^-19 T + 2^-20 of itself;
* out: u |out| for its own rounding, (u_p + 2 e) sum p|v| for the rounding
  of p (to the inputs' type in a prompt, to fp16 in decode; there a p below
  2^-14 of the running maximum is off by up to 2^-25 of it instead), and
  2^-20 sum p|v| for the fp32 sums of some hundred steps;
* lse: e for the sum, 2^-22 |lse| for its own roundings;
* attention weights: p off by 2^-18 (1 + |lse| + T) of itself (the score
  and lse enter one subtraction);
* the cache's bytes and scales, kept positions: equal.
"""
import math

import numpy as np
import pytest
import torch

from oracle import gqa_oracle as G

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def f64(t):
    return t.detach().cpu().double().numpy()


def close(got, want, tol):
    """Equal where not finite, else within tol."""
    fin = np.isfinite(want)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    np.testing.assert_array_equal(got[np.isinf(want)], want[np.isinf(want)])
    bad = np.abs(got - want)[fin] > tol[fin]
    assert not bad.any(), (np.abs(got - want)[fin][bad].max(), tol[fin][bad].min(), int(bad.sum()), int(fin.sum()))


def status():
    from deepseek_v4_kernel import gqa
    return gqa.gqa_status()


# ------------------------------------------------------------------ prompts
def check_prefill(q, k, v, cu_q, cu_k, causal, scale=None, out=None, known=None):
    import deepseek_v4_kernel as dk
    scale = q.shape[2] ** -0.5 if scale is None else scale
    cq = torch.tensor(cu_q, dtype=torch.int32, device="cuda")
    ck = None if cu_k is None else torch.tensor(cu_k, dtype=torch.int32, device="cuda")
    got, lse = dk.gqa_prefill_fwd(q, k, v, cq, ck, sm_scale=scale, causal=causal, out=out)
    torch.cuda.synchronize()
    assert status() == 0
    want, wl, mag, size = known or G.prefill(f64(q), f64(k), f64(v), cu_q, cu_q if cu_k is None else cu_k, scale, causal)
    u, n = U[q.dtype], cu_q[-1]
    e = 2.0 ** -19 * size + 2.0 ** -20
    close(f64(got)[:n], want[:n], u * np.abs(want[:n]) + ((u + 2.0 ** -20 + 2 * e)[..., None] * mag)[:n] + 1e-30)
    close(f64(lse)[:n], wl[:n], (e + 2.0 ** -22 * np.abs(np.where(np.isfinite(wl), wl, 0)))[:n])
    return got, lse


def packed(lens):
    return [0] + list(np.cumsum(lens))


def rand(g, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


@pytest.mark.parametrize("dqk,dv", [(64, 64), (128, 128), (192, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,h,hkv", [([1], 1, 1), ([5, 1, 130], 4, 2), ([128, 256, 127], 5, 1),
                                        ([129, 0, 255, 1, 257], 6, 3), ([700], 2, 2)])
def test_prefill(dqk, dv, dtype, lens, h, hkv):
    g = torch.Generator(device="cuda").manual_seed(sum(lens) + h)
    n = sum(lens)
    q, k, v = (rand(g, n, a, b, dtype=dtype) for a, b in ((h, dqk), (hkv, dqk), (hkv, dv)))
    check_prefill(q, k, v, packed(lens), None, True)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("qs,ks", [([1, 1, 1], [300, 1, 128]), ([200, 64], [513, 64]), ([130, 3, 260], [100, 0, 259]),
                                   ([40, 300], [0, 0]), ([256, 256], [384, 257])])
def test_prefill_other_key_lengths(causal, qs, ks):
    """Keys of an earlier prefix, fewer keys than queries (rows that see
    nothing), and none at all."""
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = rand(g, sum(qs), 4, 128), rand(g, sum(ks), 2, 128), rand(g, sum(ks), 2, 128)
    _, lse = check_prefill(q, k, v, packed(qs), packed(ks), causal)
    if sum(ks) == 0:
        assert torch.isneginf(lse).all()


@pytest.mark.parametrize("magnitude", [0.01, 8.0])
def test_prefill_scores_of_all_sizes(magnitude):
    """Nearly equal scores, and ones whose running maximum grows again and again."""
    g = torch.Generator(device="cuda").manual_seed(4)
    n = 900
    ramp = torch.linspace(0.1, 1, n, device="cuda")[:, None, None]
    q, k = rand(g, n, 2, 128) * magnitude, (torch.randn(n, 1, 128, generator=g, device="cuda") * ramp).bfloat16()
    check_prefill(q, k, rand(g, n, 1, 128), [0, n], None, True, scale=0.3)


def test_prefill_strides_out_and_rows_behind():
    """q, k, v as parts of one projection, a strided out, and rows behind the
    last sequence, which stay as they were."""
    g = torch.Generator(device="cuda").manual_seed(5)
    lens, h, hkv, d = [70, 200], 4, 2, 128
    n, more = sum(lens), 9
    x = rand(g, n + more, (h + 2 * hkv) * d + 8)
    x[n:] = float("nan")
    q = x[:, :h * d].unflatten(1, (h, d))
    k = x[:, h * d:(h + hkv) * d].unflatten(1, (hkv, d))
    v = x[:, (h + hkv) * d:(h + 2 * hkv) * d].unflatten(1, (hkv, d))
    base = torch.full((n + more, h, d + 8), 7.0, dtype=torch.bfloat16, device="cuda")
    check_prefill(q, k, v, packed(lens), None, True, out=base[..., :d])
    assert (base[n:] == 7.0).all() and (base[..., d:] == 7.0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_prefill_values_that_are_not_finite(what, dtype):
    """NaN and infinities reach the rows that see them and no other: not
    those before them, not those of the sequences beside theirs."""
    g = torch.Generator(device="cuda").manual_seed(6)
    lens = [150, 333, 90]
    n = sum(lens)
    q, k, v = rand(g, n, 2, 128, dtype=dtype), rand(g, n, 1, 128, dtype=dtype), rand(g, n, 1, 128, dtype=dtype)
    v[150 + 300, 0, 5] = what          # seen by its sequence's rows 300 ..
    v[150 + 200, 0, 77:80] = what
    v[483:486] = what                  # the whole third sequence sees these
    k[20, 0] = float("nan")            # rows 20 .. of the first sequence
    check_prefill(q, k, v, packed(lens), None, True)


def test_prefill_bad_offsets_stay_in_bounds():
    """cu_seqlens that run past the tensors or backwards: no row outside them
    is read or written."""
    import deepseek_v4_kernel as dk
    g = torch.Generator(device="cuda").manual_seed(7)
    q, k, v = rand(g, 300, 2, 64), rand(g, 300, 2, 64), rand(g, 300, 2, 64)
    for cu in ([0, 100, 5000], [0, 200, 100, 300], [-50, 100, 300], [300, 0, 300]):
        dk.gqa_prefill_fwd(q, k, v, torch.tensor(cu, dtype=torch.int32, device="cuda"))
        torch.cuda.synchronize()
    assert status() == 0
    check_prefill(q, k, v, [0, 300], None, True)


def test_prefill_many_sequences():
    g = torch.Generator(device="cuda").manual_seed(8)
    lens = [(7 * i) % 23 for i in range(800)]
    n = sum(lens)
    q, k, v = rand(g, n, 1, 64), rand(g, n, 1, 64), rand(g, n, 1, 64)
    check_prefill(q, k, v, packed(lens), None, True)


def test_prefill_offsets_past_32_bits():
    """q, k, v and out of more than 2^31 elements: 90,000 tokens of 128 heads
    of 192, in sequences of 200 (the last one looked at, and one in between)."""
    import deepseek_v4_kernel as dk
    g = torch.Generator(device="cuda").manual_seed(7)
    n, h, step = 90_000, 128, 200
    q = torch.randn(n, h, 192, generator=g, device="cuda", dtype=torch.bfloat16)
    k = torch.randn(n, h, 192, generator=g, device="cuda", dtype=torch.bfloat16)
    v = torch.randn(n, h, 192, generator=g, device="cuda", dtype=torch.bfloat16)[..., 64:]
    cu = torch.arange(0, n + 1, step, dtype=torch.int32, device="cuda")
    out = torch.empty(n, h, 192, device="cuda", dtype=torch.bfloat16)[..., :128]
    got, lse = dk.gqa_prefill_fwd(q, k, v, cu, out=out)
    for at in (87_400, n - step):
        part = [t[at:at + step, 125:].contiguous() for t in (q, k, v)]
        one, one_lse = check_prefill(*part, [0, step], None, True)
        assert torch.equal(got[at:at + step, 125:], one) and torch.equal(lse[at:at + step, 125:], one_lse)


# ------------------------------------------------------------------ the cache
class Cache:
    """Random pages for sequences of the given lengths; rows that hold no
    position are NaN, their blocks' scales too where no row is held."""

    def __init__(self, lens, page, hkv, d, seed, spare=2, heads_first=False, width=None):
        g = torch.Generator().manual_seed(seed)
        counts = [-(-n // page) for n in lens]
        nb = sum(counts) + spare
        self.page = page
        self.table = torch.full((len(lens), width or max(counts + [1]) + 1), -1, dtype=torch.int32)
        perm = torch.randperm(nb, generator=g)
        at = 0
        used = torch.zeros(nb, page, dtype=torch.bool)
        for i, (n, c) in enumerate(zip(lens, counts)):
            self.table[i, :c] = perm[at:at + c]
            used[perm[at:at + c]] = (torch.arange(c * page) < n).view(c, page)
            at += c
        self.free = perm[at:]
        make = []
        for _ in range(2):
            x = (torch.randn(nb, page, hkv, d, generator=g) * 60).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
            x[~used] = 0x7F
            s = torch.exp2(torch.randint(-8, -4, (nb, hkv), generator=g).float())
            s[~used.any(1)] = float("nan")
            if heads_first:
                x = x.transpose(1, 2).contiguous().transpose(1, 2)
            make += [x, s]
        self.kc, self.ks, self.vc, self.vs = make
        self.ctx = torch.tensor(lens, dtype=torch.int32)

    def cuda(self):
        """k_cache, v_cache, k_scale, v_scale, block_table, context_lens."""
        def dev(x):
            y = torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device="cuda")
            return y.copy_(x)
        return dev(self.kc).view(torch.float8_e4m3fn), dev(self.vc).view(torch.float8_e4m3fn), self.ks.cuda(), \
            self.vs.cuda(), self.table.cuda(), self.ctx.cuda()

    def np(self):
        return self.kc.numpy(), self.vc.numpy(), self.ks.numpy(), self.vs.numpy(), self.table.numpy(), self.ctx.numpy()


def check_decode(c, q, scale=None, dev=None, out=None):
    import deepseek_v4_kernel as dk
    scale = q.shape[3] ** -0.5 if scale is None else scale
    got, lse = dk.gqa_decode_fwd(q, *(dev or c.cuda()), sm_scale=scale, out=out)
    torch.cuda.synchronize()
    assert status() == 0
    kc, vc, ks, vs, table, ctx = c.np()
    want, wl, mag, size, vsum = G.decode(f64(q), kc, vc, ks, vs, table, ctx, scale)
    u = U[q.dtype]
    e = 2.0 ** -19 * size + 2.0 ** -20
    eo = np.transpose(e, (0, 2, 1))[..., None]
    close(f64(got), want, u * np.abs(want) + (2.0 ** -11 + 2.0 ** -20 + 2 * eo) * mag + 2.0 ** -25 * vsum + 1e-30)
    close(f64(lse), wl, e + 2.0 ** -22 * np.abs(np.where(np.isfinite(wl), wl, 0)))
    return got, lse


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 256])
@pytest.mark.parametrize("lens", [[1], [31, 32, 33, 0, 64], [500, 7, 130]])
def test_decode(d, page, lens):
    g = torch.Generator(device="cuda").manual_seed(d + page)
    c = Cache(lens, page, 2, d, seed=page)
    check_decode(c, rand(g, len(lens), 1, 8, d))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("h,hkv,sq", [(1, 1, 1), (3, 3, 2), (12, 1, 1), (16, 2, 3), (40, 2, 1), (24, 1, 5), (5, 1, 40)])
def test_decode_heads_and_drafts(h, hkv, sq, dtype):
    """Rows up to many groups of 16, queries that see different positions,
    sequences shorter than the drafts (rows that see nothing)."""
    g = torch.Generator(device="cuda").manual_seed(h + sq)
    for d, page in ((128, 32), (64, 16)):
        c = Cache([70, 1, 0, 33, 260], page, hkv, d, seed=h)
        check_decode(c, rand(g, 5, sq, h, d, dtype=dtype))


def test_decode_long_is_shared_by_all_sms():
    g = torch.Generator(device="cuda").manual_seed(2)
    for d, hkv, lens in ((128, 1, [20000]), (64, 2, [9000, 3, 5000])):
        c = Cache(lens, 64, hkv, d, seed=3)
        check_decode(c, rand(g, len(lens), 1, 4 * hkv, d) * 3)


def test_decode_many_sequences():
    g = torch.Generator(device="cuda").manual_seed(2)
    lens = [(37 * i) % 90 for i in range(600)]
    c = Cache(lens, 16, 1, 64, seed=3)
    check_decode(c, rand(g, len(lens), 1, 2, 64))


@pytest.mark.parametrize("magnitude", [1e-3, 20.0, 1e30])
def test_decode_scales_and_magnitudes(magnitude):
    """q of any size (scaled against by sm_scale), scales of every kind:
    zero, not a power of two, far apart between blocks."""
    g = torch.Generator(device="cuda").manual_seed(9)
    c = Cache([400, 300], 16, 2, 128, seed=5)
    c.vs *= torch.exp2(torch.randint(-20, 20, c.vs.shape, generator=torch.Generator().manual_seed(1)).float()) * 1.3
    c.vs[c.table[0, 3].item()] = 0.0
    c.ks[c.table[0, 5].item()] = 0.0
    c.ks[c.table[1, 2].item()] *= 1.7
    q = (torch.randn(2, 1, 8, 128, generator=g, device="cuda") * magnitude).bfloat16()
    check_decode(c, q, scale=128 ** -0.5 / magnitude)


def test_decode_layouts_and_out():
    """Heads before rows in a page, a padded pool, strided q and out, one
    sequence's blocks anywhere."""
    g = torch.Generator(device="cuda").manual_seed(10)
    c = Cache([100, 222], 32, 4, 128, seed=6, heads_first=True)
    q = rand(g, 2, 2, 8, 136)[..., :128]
    base = torch.full((2, 2, 8, 160), 3.0, dtype=torch.bfloat16, device="cuda")
    check_decode(c, q, out=base[..., :128])
    assert (base[..., 128:] == 3.0).all()
    kc, vc, *rest = c.cuda()
    pad = torch.zeros(kc.shape[0] + 1, 2, 32, 4, 144, dtype=torch.uint8, device="cuda")
    pad[1:, 0, :, :, :128], pad[1:, 1, :, :, :128] = kc.view(torch.uint8), vc.view(torch.uint8)
    check_decode(c, q, dev=(pad[1:, 0, :, :, :128], pad[1:, 1, :, :, :128], *rest))


@pytest.mark.parametrize("page", [16, 64])
def test_decode_bad_blocks_hold_nothing(page):
    g = torch.Generator(device="cuda").manual_seed(11)
    c = Cache([300, 90, 20], page, 2, 128, seed=7)
    c.table[0, 1] = -1
    c.table[0, 3] = c.kc.shape[0]
    c.table[2, :] = 2 ** 31 - 1
    out, lse = check_decode(c, rand(g, 3, 2, 4, 128))
    assert (out[2] == 0).all() and torch.isneginf(lse[2]).all()
    # a table narrower than the context: what lies past it is not there
    c = Cache([page * 3, page], page, 2, 128, seed=8)
    c.ctx[0] = page * 9
    check_decode(c, rand(g, 2, 1, 4, 128))


def test_decode_nan_is_seen_only_by_those_who_see_it():
    g = torch.Generator(device="cuda").manual_seed(12)
    c = Cache([64, 45], 32, 1, 128, seed=9)
    for i, t in ((0, 63), (0, 62), (1, 44)):          # the last drafts' own positions
        blk = c.table[i, t // 32].item()
        c.vc[blk, t % 32, 0, 3 + t % 5] = 0x7F
    blk = c.table[1, 1].item()
    c.kc[blk, 43 % 32, 0, 0] = 0xFF
    out, _ = check_decode(c, rand(g, 2, 3, 4, 128))
    assert torch.isfinite(out[0, 0]).all() and torch.isfinite(out[1, 0]).all() and torch.isnan(out[0, 2]).any()


@pytest.mark.parametrize("lens", [[1, 40], [3000, 200]])
def test_decode_nan_queries(lens):
    """A query whose scores are all NaN gets NaN, its neighbours in the tile nothing of it."""
    g = torch.Generator(device="cuda").manual_seed(13)
    c = Cache(lens, 64, 1, 128, seed=10)
    q = rand(g, 2, 1, 6, 128)
    q[0, 0, 1, 7], q[1, 0, 4, 100] = float("nan"), float("inf")
    out, lse = check_decode(c, q)
    assert torch.isnan(out[0, 0, 1]).all() and torch.isnan(lse[0, 1, 0]) and int(torch.isnan(out).any(-1).sum()) == 2


def test_decode_and_weights_far_into_a_pool():
    """Blocks whose bytes lie past 2^32 of the pool, the tensors' strides included."""
    import deepseek_v4_kernel as dk
    g = torch.Generator(device="cuda").manual_seed(14)
    c = Cache([200, 100], 64, 2, 128, seed=11, spare=0)
    used, far = c.kc.shape[0], 300_000  # of 16 KB
    big = [torch.empty(far + used, 64, 2, 128, dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = [torch.empty(far + used, 2, device="cuda") for _ in range(2)]
    for t, x in zip(big + scales, (c.kc, c.vc, c.ks, c.vs)):
        t[far:] = x.cuda()
    table = torch.where(c.table >= 0, c.table + far, c.table).cuda()
    q, near = rand(g, 2, 2, 8, 128), c.cuda()
    res = []
    for kc, vc, ks, vs, tab in ((*near[:4], near[4]), (*big, *scales, table)):
        o, lse = dk.gqa_decode_fwd(q, kc, vc, ks, vs, tab, near[5])
        res.append((o, lse, dk.gqa_attention_weights(q, lse, kc, ks, tab, near[5])))
    for x, y in zip(*res):
        assert torch.equal(x, y)
    # and written there
    k, v = rand(g, 70, 2, 128), rand(g, 70, 2, 128)
    cu, ctx = torch.tensor([0, 10, 70], dtype=torch.int32, device="cuda"), torch.tensor([200, 100], dtype=torch.int32, device="cuda")
    dk.gqa_cache_append(k, v, cu, ctx, near[4], *near[:4])
    dk.gqa_cache_append(k, v, cu, ctx, table, *big, *scales)
    new = torch.tensor([[0, far - 2], [far - 1, 7]], dtype=torch.int32, device="cuda")
    w = res[0][2]
    small = [torch.cat([t, torch.zeros_like(t[:4])]) for t in (x.view(torch.uint8) if x.element_size() == 1 else x for x in near[:4])]
    new_near = torch.arange(used, used + 4, dtype=torch.int32, device="cuda").view(2, 2)
    got = dk.gqa_cache_evict(*big, *scales, table, near[5], w, 90, 20, new)
    want = dk.gqa_cache_evict(*small, near[4], near[5], w, 90, 20, new_near)
    for x, y in zip(got, want):
        assert torch.equal(x, y)
    for t, x, y in zip(big + scales, small, near[:4]):
        y = y.view(torch.uint8) if y.element_size() == 1 else y
        assert torch.equal(t[far:].view(torch.uint8), y.view(torch.uint8))
        for i in range(2):
            a, b = t[new[i].long()].flatten(0, 1), x[new_near[i].long()].flatten(0, 1)
            n = 90 if t.dim() == 4 else len(a)
            assert torch.equal(a[:n].view(torch.uint8), b[:n].view(torch.uint8))
    torch.cuda.synchronize()
    assert status() == 0


# ------------------------------------------------------------------ weights
def check_weights(c, q, width=None, into=None, accumulate=False, lse=None):
    import deepseek_v4_kernel as dk
    kc, vc, ks, vs, table, ctx = dev = c.cuda()
    if lse is None:
        _, lse = dk.gqa_decode_fwd(q, *dev)
    before = None if into is None else into.clone()
    got = dk.gqa_attention_weights(q, lse, kc, ks, table, ctx, weights=into, accumulate=accumulate, max_context=width)
    torch.cuda.synchronize()
    assert status() == 0
    n = c.np()
    want, e = G.weights(f64(q), f64(lse), n[0], n[2], n[4], n[5], q.shape[3] ** -0.5, got.shape[2])
    tol = 2.0 ** -18 * e + 1e-30
    if accumulate:
        want = want + f64(before)
        tol = tol + 2.0 ** -23 * np.abs(want)
    close(f64(got), want, tol)
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("h,hkv,sq,d,page", [(4, 1, 1, 128, 64), (16, 2, 1, 64, 16), (8, 2, 7, 128, 16),
                                             (12, 1, 40, 64, 32), (6, 2, 100, 128, 32)])
def test_weights(h, hkv, sq, d, page, dtype):
    """One group of rows up to more groups than are held at once."""
    g = torch.Generator(device="cuda").manual_seed(h + sq)
    c = Cache([300, 0, 1, 97, 128], page, hkv, d, seed=h)
    w = check_weights(c, rand(g, 5, sq, h, d, dtype=dtype))
    assert (w[1] == 0).all()
    live = c.ctx >= sq
    total = w.sum(2).cpu()[live]
    torch.testing.assert_close(total, torch.full_like(total, h // hkv * sq), rtol=2e-4, atol=0)


@pytest.mark.parametrize("h,hkv,sq,d", [(1, 1, 9, 64), (4, 2, 40, 128), (4, 2, 100, 64), (4, 1, 90, 128), (8, 2, 1, 128)])
def test_weights_many_units_of_every_cta(h, hkv, sq, d):
    """One row up to more than are held at once, over contexts that wrap every
    ring; the 64-bit sums on the GPU (tolerances as in check_weights)."""
    import deepseek_v4_kernel as dk
    g = torch.Generator(device="cuda").manual_seed(sq)
    c = Cache([130000, 63, 70001], 256, hkv, d, seed=h)
    kc, vc, ks, vs, table, ctx = dev = c.cuda()
    q = rand(g, 3, sq, h, d)
    _, lse = dk.gqa_decode_fwd(q, *dev)
    got = dk.gqa_attention_weights(q, lse, kc, ks, table, ctx)
    for i, n in enumerate(c.ctx.tolist()):
        t = torch.arange(n, device="cuda")
        blk = table[i, t // 256].long()
        assert (got[i, :, n:] == 0).all()
        for kvh in range(hkv):
            k = kc[blk, t % 256, kvh].double() * ks[blk, kvh].double()[:, None]
            want, tol = torch.zeros(n, device="cuda", dtype=torch.float64), torch.zeros(n, device="cuda", dtype=torch.float64)
            for x in range(sq):
                rows = q[i, x, kvh * (h // hkv):(kvh + 1) * (h // hkv)].double()
                row_lse = lse[i, kvh * (h // hkv):(kvh + 1) * (h // hkv), x].double()[:, None]
                p = torch.exp(rows @ k.T * d ** -0.5 - row_lse)
                p = torch.where((t <= n - sq + x) & torch.isfinite(row_lse), p, 0)
                want += p.sum(0)
                tol += (p * (1 + row_lse.abs() + rows.abs() @ k.abs().T * d ** -0.5)).nan_to_num(0, 0, 0).sum(0)
            assert ((got[i, kvh, :n].double() - want).abs() <= 2.0 ** -18 * tol + 1e-30).all()
    torch.cuda.synchronize()
    assert status() == 0


def test_weights_rows_of_many_sizes():
    """Rows of q whose magnitudes lie far apart, beside equal ones, and rows of zeros."""
    g = torch.Generator(device="cuda").manual_seed(3)
    c = Cache([500, 129], 64, 2, 128, seed=5)
    q = rand(g, 2, 40, 4, 128)
    q *= torch.exp2(torch.randint(-12, 2, (2, 40, 4, 1), generator=g, device="cuda").float()).bfloat16()
    q[0, :, :, :] = rand(g, 40, 4, 128)
    q[0, 20:, 1] = 0
    q[1, 30:, 3] = 0
    check_weights(c, q)


def test_weights_into_a_tensor():
    g = torch.Generator(device="cuda").manual_seed(1)
    c = Cache([200, 90], 32, 2, 128, seed=2)
    q = rand(g, 2, 1, 8, 128)
    store = torch.full((2, 2, 300), 5.0, device="cuda")
    w = check_weights(c, q, into=store[..., :250])
    assert w.data_ptr() == store.data_ptr() and (store[..., 250:] == 5.0).all() and (store[1, :, 90:250] == 0).all()
    store.fill_(5.0)
    check_weights(c, q, into=store, accumulate=True)
    assert (store[1, :, 90:] == 5.0).all()
    # narrower than the context: the rest is left out
    assert check_weights(c, q, width=130).shape[2] == 130


def test_weights_bad_blocks_and_empty_rows():
    g = torch.Generator(device="cuda").manual_seed(2)
    c = Cache([200, 2], 32, 2, 64, seed=3)
    c.table[0, 2] = -5
    w = check_weights(c, rand(g, 2, 4, 8, 64))
    assert (w[0, :, 64:96] == 0).all()


# ------------------------------------------------------------------ append
def check_append(c, x, cu, ctx, dtype):
    import deepseek_v4_kernel as dk
    c.ctx = torch.tensor(ctx, dtype=torch.int32)
    kc, vc, ks, vs, table, ctx_d = c.cuda()
    k, v = x
    dk.gqa_cache_append(k, v, torch.tensor(cu, dtype=torch.int32, device="cuda"), ctx_d, table, kc, vc, ks, vs)
    torch.cuda.synchronize()
    n = c.np()
    for t, i in ((k, 0), (v, 1)):
        G.append(f64(t), cu, ctx, n[4], n[i], n[2 + i])
    for got, want in ((kc, n[0]), (vc, n[1])):
        g = got.view(torch.uint8).cpu().numpy()
        same = (g == want) | (((g & 0x7F) == 0x7F) & ((want & 0x7F) == 0x7F))
        assert same.all(), np.argwhere(~same)[:5]
    np.testing.assert_array_equal(ks.cpu().numpy(), n[2])
    np.testing.assert_array_equal(vs.cpu().numpy(), n[3])
    return kc, vc, ks, vs, table, ctx_d


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("old,new", [([0], [1]), ([0, 15, 16, 17, 63, 64], [1, 1, 1, 1, 1, 1]),
                                     ([3, 0, 100, 5, 0], [200, 0, 29, 1, 500])])
def test_append(dtype, d, page, old, new):
    g = torch.Generator(device="cuda").manual_seed(page + d)
    ctx = [a + b for a, b in zip(old, new)]
    c = Cache(old, page, 3, d, seed=page, spare=len(old) + sum(-(-n // page) for n in ctx), width=-(-max(ctx) // page) + 1)
    free = iter(c.free.tolist())
    for i, n in enumerate(ctx):
        for p in range(-(-n // page)):
            if c.table[i, p] < 0:
                c.table[i, p] = next(free)
    size = torch.exp(torch.randn(sum(new), 1, 1, generator=g, device="cuda") * 2)
    x = [(torch.randn(sum(new), 3, d, generator=g, device="cuda") * size).to(dtype) for _ in range(2)]
    check_append(c, x, packed(new), ctx, dtype)


def test_append_odd_values():
    """Zeros, infinities, NaN, the smallest and largest values, scales that
    grow by steps that round the older rows, a scale that is no power of
    two, rows of strided tensors, blocks that are not there."""
    g = torch.Generator(device="cuda").manual_seed(3)
    c = Cache([10, 20, 0, 40], 32, 2, 64, seed=4, spare=8, width=3)
    free = iter(c.free.tolist())
    ctx = [12, 40, 33, 70]
    for i, n in enumerate(ctx):
        for p in range(-(-n // 32)):
            if c.table[i, p] < 0:
                c.table[i, p] = next(free)
    c.table[3, 2] = -1
    blk = c.table[1, 0].item()
    c.ks[blk], c.vs[blk] = 0.3, 1e-20
    new = [2, 20, 33, 30]
    n = sum(new)
    big = torch.randn(n, 5, 2, 64 + 8, generator=g, device="cuda").bfloat16()
    k, v = big[:, 1, :, :64], big[:, 3, :, :64]
    k[0] *= 1000
    v[0] = 0
    v[1] = 0
    k[1, 0, 3], k[1, 1, 4], k[5, 0, 6] = float("inf"), -float("inf"), float("nan")
    v[30] = 3.3e38
    k[31] = 1e-38
    k[22:55, 1] = 0
    v[22:55, 0] = 1e-37
    check_append(c, (k, v), packed(new), ctx, torch.bfloat16)


def test_append_tokens_before_position_zero_and_rows_behind():
    """A context shorter than its new tokens: the first ones are skipped.
    Rows behind the last sequence are not stored."""
    g = torch.Generator(device="cuda").manual_seed(4)
    c = Cache([0, 0], 16, 1, 64, seed=4, spare=6, width=2)
    c.table[0, 0], c.table[1, 0], c.table[1, 1] = c.free[:3].tolist()
    x = [rand(g, 50, 1, 64) for _ in range(2)]
    check_append(c, x, [0, 20, 40], [5, 20], torch.bfloat16)


# ------------------------------------------------------------------ eviction
def check_evict(c, w, budget, recent, new_width=None):
    import deepseek_v4_kernel as dk
    dev = c.cuda()
    b, hkv = w.shape[:2]
    blocks = -(-budget // c.page)
    new_table = torch.full((b, blocks), -1, dtype=torch.int32)
    free = iter(c.free.tolist())
    for i in range(b):
        for p in range(-(-min(int(c.ctx[i]), budget) // c.page)):
            new_table[i, p] = next(free)
    into = None if new_width is None else torch.full((b, hkv, new_width), 9.0, device="cuda")
    kept, nw, lens = dk.gqa_cache_evict(*dev, w.cuda(), budget, recent, new_table.cuda(), new_weights=into)
    torch.cuda.synchronize()
    n = c.np()
    want, ww, wl = G.evict(*n, w.numpy(), budget, recent, new_table.numpy())
    np.testing.assert_array_equal(kept.cpu().numpy(), want)
    np.testing.assert_array_equal(nw.cpu().numpy()[..., :budget], ww)
    assert (nw.cpu().numpy()[..., budget:] == 0).all()
    np.testing.assert_array_equal(lens.cpu().numpy(), wl)
    for i in range(2):
        g = dev[i].view(torch.uint8).cpu().numpy()
        same = (g == n[i]) | (((g & 0x7F) == 0x7F) & ((n[i] & 0x7F) == 0x7F))
        assert same.all(), np.argwhere(~same)[:5]
        np.testing.assert_array_equal(dev[2 + i].cpu().numpy(), n[2 + i])
    return kept


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("lens,budget,recent", [([1], 1, 0), ([300, 5, 64, 0, 128], 64, 16), ([2500, 77], 1000, 1000),
                                                ([5000], 700, 0), ([90, 91], 90, 89)])
def test_evict(d, page, lens, budget, recent):
    g = torch.Generator().manual_seed(page)
    need = sum(-(-min(n, budget) // page) for n in lens)
    c = Cache(lens, page, 2, d, seed=d, spare=need + 1)
    w = torch.randn(len(lens), 2, max(lens) + 3, generator=g).exp()
    check_evict(c, w, budget, recent)


@pytest.mark.parametrize("kind", ["all equal", "few values", "signs", "nan and inf"])
def test_evict_ties(kind):
    g = torch.Generator().manual_seed(1)
    c = Cache([3000, 700], 64, 2, 64, seed=3, spare=30)
    w = torch.randn(2, 2, 3000, generator=g)
    if kind == "all equal":
        w = torch.zeros_like(w)
    elif kind == "few values":
        w = (w * 2).round().abs()
    elif kind == "signs":
        w = (w * 4).round() / 4 * torch.where(torch.rand(w.shape, generator=g) < 0.5, 1.0, -1.0)  # -0.0 and 0.0
    else:
        w[torch.rand(w.shape, generator=g) < 0.1] = float("nan")
        w[torch.rand(w.shape, generator=g) < 0.1] = float("inf")
        w[torch.rand(w.shape, generator=g) < 0.1] = -float("inf")
    c.vs *= 1.37  # scales that are no powers of two
    check_evict(c, w, 500, 20, new_width=640)


def test_evict_bad_blocks_and_narrow_weights():
    g = torch.Generator().manual_seed(2)
    c = Cache([400, 300], 32, 2, 128, seed=3, spare=14)
    c.table[0, 3] = -1
    c.table[1, 0] = 10 ** 6
    check_evict(c, torch.rand(2, 2, 320, generator=g), 200, 10)  # width 320: the first counts as 320 long


# ------------------------------------------------------------------ together
def test_a_serving_run():
    """Prompts -> cache -> decode with drafts -> weights -> eviction ->
    further decode over what is left, against the oracle at every step."""
    import deepseek_v4_kernel as dk
    g = torch.Generator(device="cuda").manual_seed(20)
    lens, h, hkv, d, page, budget = [200, 45, 131], 8, 2, 128, 32, 96
    b, n = len(lens), sum(lens)
    qkv = rand(g, n, (h + 2 * hkv) * d)
    q, k, v = (x.unflatten(1, (-1, d)) for x in qkv.split([h * d, hkv * d, hkv * d], dim=1))
    check_prefill(q, k, v, packed(lens), None, True)

    c = Cache([0] * b, page, hkv, d, seed=1, spare=60, width=8)
    ids = iter(c.free.tolist())
    c.table[:] = torch.tensor([[next(ids) for _ in range(8)] for _ in range(b)])
    dev = check_append(c, (k, v), packed(lens), lens, torch.bfloat16)
    # drafts: their keys go in first, then they attend
    s_q = 3
    for _ in range(2):
        lens = [x + s_q for x in lens]
        kn, vn = rand(g, b * s_q, hkv, d), rand(g, b * s_q, hkv, d)
        dev = check_append(c, (kn, vn), packed([s_q] * b), lens, torch.bfloat16)
        qn = rand(g, b, s_q, h, d)
        check_decode(c, qn, dev=dev)
    w = check_weights(c, qn)
    c.free = torch.tensor([next(ids) for _ in range(b * 3)])
    new = c.free.view(b, 3).int()
    kept = check_evict(c, w.cpu(), budget, 20)
    # the kept positions alone, from the new blocks
    counts = [-(-min(x, budget) // page) for x in lens]
    at = 0
    table = torch.full((b, 3), -1, dtype=torch.int32)
    for i, m in enumerate(counts):
        table[i, :m] = c.free[at:at + m]
        at += m
    c.table, c.ctx = table, torch.tensor([min(x, budget) for x in lens], dtype=torch.int32)
    check_decode(c, rand(g, b, 1, h, d))
    assert (kept >= 0).sum() == hkv * int(c.ctx.sum())


@pytest.mark.parametrize("page", [512, 1024])
def test_large_pages(page):
    """Every operator over the largest blocks: whole, cut short, and shared by old and new rows."""
    g = torch.Generator(device="cuda").manual_seed(21)
    old, new = [page - 1, 0, 700], [600, 3, page]
    c = Cache(old, page, 2, 128, seed=4, spare=12, width=3)
    for i in range(3):  # room for the new ones
        have = -(-old[i] // page)
        want = -(-(old[i] + new[i]) // page)
        c.table[i, have:want] = c.free[2 * i:2 * i + want - have]
    c.ctx = torch.tensor([x + y for x, y in zip(old, new)], dtype=torch.int32)
    kv = rand(g, sum(new), 2, 128), rand(g, sum(new), 2, 128)
    dev = check_append(c, kv, packed(new), c.ctx.tolist(), torch.bfloat16)
    q = rand(g, 3, 2, 8, 128)
    check_decode(c, q, dev=dev)
    w = check_weights(c, q[:, -1:])
    check_weights(c, rand(g, 3, 12, 8, 128))
    c.free = c.free[6:]
    check_evict(c, w.cpu(), page + 50, 64)


def test_evict_into_bad_blocks():
    """New blocks that are not there are not written, the rest is as without them."""
    import deepseek_v4_kernel as dk
    g = torch.Generator().manual_seed(22)
    c = Cache([300, 200], 32, 2, 64, seed=3, spare=8)
    w = torch.rand(2, 2, 320, generator=g).cuda()
    new = c.free[:8].int().view(2, 4).cuda()
    good, bad = c.cuda(), c.cuda()
    want = dk.gqa_cache_evict(*good, w, 100, 10, new)
    hole = new.clone()
    hole[0, 1], hole[1, 3], hole[1, 0] = -1, 2 ** 31 - 1, c.kc.shape[0]
    got = dk.gqa_cache_evict(*bad, w, 100, 10, hole)
    for x, y in zip(want, got):
        assert torch.equal(x, y)
    kept = torch.tensor([new[0, 0], new[0, 2], new[0, 3], new[1, 1], new[1, 2]], device="cuda").long()
    lost = torch.tensor([new[0, 1], new[1, 3], new[1, 0]], device="cuda").long()
    first = c.cuda()
    for i in range(4):
        x, y, z = (t[i].view(torch.uint8) for t in (good, bad, first))
        assert torch.equal(x[kept], y[kept]) and torch.equal(y[lost], z[lost])
        rest = torch.ones(len(x), dtype=torch.bool, device="cuda")
        rest[new.flatten().long()] = False
        assert torch.equal(y[rest], z[rest])
    assert status() == 0


def test_graph_streams_and_two_at_once():
    """Captured in two graphs that share nothing, replayed on two streams at
    once, with inputs that changed in place; the results are those of plain
    calls, bit for bit."""
    import deepseek_v4_kernel as dk
    g = torch.Generator(device="cuda").manual_seed(30)
    cases = []
    for seed, lens in ((1, [700, 3000, 20]), (2, [5000, 1, 900])):
        c = Cache(lens, 64, 2, 128, seed=seed, spare=0)
        dev = c.cuda()
        q = rand(g, 3, 2, 8, 128)
        x = rand(g, 400, 8, 128)
        kv = rand(g, 400, 2, 128)
        cu = torch.tensor([0, 130, 130, 400], dtype=torch.int32, device="cuda")
        cases.append((dev, q, x, kv, cu))

    def step(dev, q, x, kv, cu):
        o, lse = dk.gqa_decode_fwd(q, *dev)
        w = dk.gqa_attention_weights(q, lse, dev[0], dev[2], dev[4], dev[5])
        return (o, lse, w) + dk.gqa_prefill_fwd(x, kv, kv, cu)

    graphs = []
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for case in cases:
            step(*case)
    side.synchronize()
    for case in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            res = step(*case)
        graphs.append((graph, res))
    for case in cases:
        case[1].copy_(rand(g, *case[1].shape))
        case[2].copy_(rand(g, *case[2].shape))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        for (graph, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for case, (_, res) in zip(cases, graphs):
        for got, want in zip(res, step(*case)):
            assert torch.equal(got, want)
    torch.cuda.synchronize()
    assert status() == 0


def test_the_same_call_twice():
    """Bit for bit: no sum's order depends on who comes first."""
    import deepseek_v4_kernel as dk
    g = torch.Generator(device="cuda").manual_seed(31)
    c = Cache([9000, 40, 333], 64, 2, 128, seed=4, spare=20)
    dev, q = c.cuda(), rand(g, 3, 2, 8, 128)
    x, kv = rand(g, 1000, 8, 128), rand(g, 1000, 2, 128)
    cu = torch.tensor([0, 900, 1000, 1000], dtype=torch.int32, device="cuda")
    new = c.free[:12].int().view(3, 4).cuda()

    def run():
        o, lse = dk.gqa_decode_fwd(q, *dev)
        w = dk.gqa_attention_weights(q, lse, dev[0], dev[2], dev[4], dev[5])
        return (o, lse, w) + dk.gqa_prefill_fwd(x, kv, kv, cu) + dk.gqa_cache_evict(*dev, w, 200, 30, new)

    first = run()
    for _ in range(3):
        for a, b in zip(first, run()):
            assert torch.equal(a, b)


def test_eviction_and_append_in_a_graph():
    """A whole step of a cache that lives in a graph: append, decode, weights
    added up, eviction into other blocks."""
    import deepseek_v4_kernel as dk
    g = torch.Generator(device="cuda").manual_seed(32)
    c = Cache([150, 64], 32, 2, 64, seed=6, spare=8)
    q, k, v = rand(g, 2, 1, 4, 64), rand(g, 2, 2, 64), rand(g, 2, 2, 64)
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    new = c.free[:8].int().view(2, 4).cuda()

    def state():
        return list(c.cuda()) + [torch.zeros(2, 2, 192, device="cuda")]

    def step(kc, vc, ks, vs, table, ctx, w):
        dk.gqa_cache_append(k, v, cu, ctx, table, kc, vc, ks, vs)
        o, lse = dk.gqa_decode_fwd(q, kc, vc, ks, vs, table, ctx)
        dk.gqa_attention_weights(q, lse, kc, ks, table, ctx, weights=w, accumulate=True)
        return (o, lse) + dk.gqa_cache_evict(kc, vc, ks, vs, table, ctx, w, 100, 10, new)

    plain, held = state(), state()
    keep = [t.clone() for t in held]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(*held)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        res = step(*held)
    for t, x in zip(held, keep):
        t.copy_(x)
    for _ in range(2):  # the second step adds its weights to the first's
        want = step(*plain)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(res, want):
            assert torch.equal(a, b)
    for t, x in zip(held, plain):
        assert torch.equal(t.view(torch.uint8), x.view(torch.uint8))


# ------------------------------------------------------------------ refusals
def test_python_refusals():
    """What the Python checks refuse before anything is launched (RuntimeError)."""
    import deepseek_v4_kernel as dk
    c = Cache([70, 64], 32, 2, 128, seed=1, spare=8)
    kc, vc, ks, vs, table, ctx = dev = c.cuda()
    q = torch.zeros(2, 1, 4, 128, dtype=torch.bfloat16, device="cuda")
    new = c.free[:4].int().view(2, 2).cuda()
    w = torch.zeros(2, 2, 96, device="cuda")
    lse = torch.zeros(2, 4, 1, device="cuda")
    k = torch.zeros(3, 2, 128, dtype=torch.bfloat16, device="cuda")
    cu = torch.tensor([0, 1, 3], dtype=torch.int32, device="cuda")
    before = [t.clone() for t in dev]

    def cache(**change):
        names = ("k_cache", "v_cache", "k_scale", "v_scale", "block_table", "context_lens")
        return {**dict(zip(names, dev)), **change}

    bad_cache = [dict(k_cache=kc.view(torch.int8)), dict(k_cache=kc.cpu()), dict(v_cache=vc[:-1]), dict(k_cache=kc[..., :96], v_cache=vc[..., :96]),
                 dict(k_cache=kc[:, :24], v_cache=vc[:, :24]), dict(v_cache=vc.transpose(0, 1).contiguous().transpose(0, 1)[:, :, :1]),
                 dict(k_cache=kc[:1].expand(kc.shape)), dict(k_scale=ks.half()), dict(v_scale=vs.t().contiguous().t()),
                 dict(v_scale=vs[:-1]), dict(block_table=table.long()), dict(block_table=table[:1]), dict(block_table=table[:, ::2]),
                 dict(context_lens=ctx.long()), dict(context_lens=ctx.cpu()), dict(context_lens=ctx.repeat(2)[::2])]
    for change in bad_cache:
        args = cache(**change)
        with pytest.raises(RuntimeError):
            dk.gqa_decode_fwd(q, **args)
        with pytest.raises(RuntimeError):
            dk.gqa_cache_append(k, k, cu, **args)
        with pytest.raises(RuntimeError):
            dk.gqa_cache_evict(**args, weights=w, budget=40, recent=4, new_block_table=new)
    for bad in (q.float(), q.cpu(), q[..., :64], q[:1], q[:, :, :3], q.view(2, 4, 128), q.new_zeros(2, 1, 4, 129)[..., 1:],
                q.new_zeros(2, 1, 128, 4).transpose(2, 3)):
        with pytest.raises(RuntimeError):
            dk.gqa_decode_fwd(bad, *dev)
        with pytest.raises(RuntimeError):
            dk.gqa_attention_weights(bad, lse, kc, ks, table, ctx)
    for kw in (dict(sm_scale=0.0), dict(sm_scale=-1.0), dict(sm_scale=float("nan")), dict(out=q.half()), dict(out=q[:1]),
               dict(out=q[:, :, :1].expand(q.shape)), dict(out=q.new_zeros(2, 1, 4, 136)[..., 4:132])):
        with pytest.raises(RuntimeError):
            dk.gqa_decode_fwd(q, *dev, **kw)
    for kw in (dict(accumulate=True), dict(max_context=0), dict(weights=w, max_context=96), dict(weights=w.double()),
               dict(weights=w[:1]), dict(weights=w[:, :, ::2]), dict(weights=w[:, :1].expand(w.shape))):
        with pytest.raises(RuntimeError):
            dk.gqa_attention_weights(q, lse, kc, ks, table, ctx, **kw)
    for bad in (lse.half(), lse[:, :2], lse.cpu(), lse.transpose(1, 2).contiguous().transpose(1, 2).expand(2, 4, 1)[:1]):
        with pytest.raises(RuntimeError):
            dk.gqa_attention_weights(q, bad, kc, ks, table, ctx)
    for kw in (dict(k=k.float()), dict(v=k[:2]), dict(v=k.half()), dict(k=k[:, :1], v=k[:, :1]), dict(k=k.cpu()), dict(cu_seqlens=cu[:2]),
               dict(cu_seqlens=cu.long())):
        with pytest.raises(RuntimeError):
            dk.gqa_cache_append(**{**dict(k=k, v=k, cu_seqlens=cu), **kw}, **cache())
    for kw in (dict(budget=0), dict(recent=41), dict(recent=-1), dict(budget=65), dict(new_block_table=table), dict(new_block_table=new[:1]),
               dict(new_weights=w), dict(new_weights=w[:, :, 1:40]), dict(weights=w.half()), dict(new_weights=w.clone()[:, :1].expand(w.shape))):
        with pytest.raises(RuntimeError):
            dk.gqa_cache_evict(*dev, **{**dict(weights=w, budget=40, recent=4, new_block_table=new), **kw})
    x, y = torch.zeros(9, 4, 128, dtype=torch.bfloat16, device="cuda"), torch.zeros(9, 2, 128, dtype=torch.bfloat16, device="cuda")
    cx = torch.tensor([0, 9], dtype=torch.int32, device="cuda")
    for args in ((x, y, y[:8], cx), (x, y.half(), y, cx), (x.float(), y.float(), y.float(), cx), (x[..., :96], y[..., :96], y[..., :96], cx),
                 (x[:, :3], y, y, cx), (x, y, y, cx[:1]), (x, y, y, cx.long()), (x, y[:5], y[:5], cx), (x[:1].expand(x.shape), y, y, cx),
                 (x, y[:, :1].expand(y.shape), y, cx), (x, y, y, cx.cpu()), (x[..., :64], y[..., :64], y, cx)):
        with pytest.raises(RuntimeError):
            dk.gqa_prefill_fwd(*args)
    for kw in (dict(out=x.half()), dict(out=x[:5]), dict(sm_scale=float("inf")), dict(out=x[:1].expand(x.shape))):
        with pytest.raises(RuntimeError):
            dk.gqa_prefill_fwd(x, y, y, cx, **kw)
    torch.cuda.synchronize()
    for t, old in zip(dev, before):  # nothing was written
        assert torch.equal(t.view(torch.uint8), old.view(torch.uint8))
    assert status() == 0


@pytest.mark.parametrize("which", ["prefill", "decode"])
def test_a_wait_that_runs_out_then_recovers(which):
    """The first load of every CTA withheld: its wait gives up after about 2 s,
    the kernel ends by itself, the status word says so, and the next call is right."""
    import deepseek_v4_kernel as dk
    from deepseek_v4_kernel import _lib
    g = torch.Generator(device="cuda").manual_seed(33)
    c = Cache([700, 90], 64, 2, 128, seed=2)
    dev, q = c.cuda(), rand(g, 2, 1, 8, 128)
    x, kv = rand(g, 600, 4, 128), rand(g, 600, 2, 128)
    cu = torch.tensor([0, 450, 600], dtype=torch.int32, device="cuda")

    def run():
        return dk.gqa_prefill_fwd(x, kv, kv, cu) if which == "prefill" else dk.gqa_decode_fwd(q, *dev)

    run()
    assert status() == 0
    try:
        assert _lib.lib.dsv4b_set_test_stall(_lib.STALL_GQA) == 0
        run()
        torch.cuda.synchronize()
        assert status() == 1
    finally:
        assert _lib.lib.dsv4b_set_test_stall(0) == 0
    assert status() == 0
    if which == "prefill":
        check_prefill(x, kv, kv, [0, 450, 600], None, True)
    else:
        check_decode(c, q, dev=dev)
