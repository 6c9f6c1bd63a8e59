"""Errors of attention over the 4-bit KV cache against 64 bits, relative to the terms that are summed (the bounds of
test_gpu_kv4.py go by the largest value of a head).

With p the softmax weights, v the values and e s a value's distance from its group's middle:
  a score is off by ds <= 16 U sum |q k| scale (f32 sums of up to 256 products, whatever the inputs' type), which moves an
      output by 2 ds sum p |v| at most, and by nothing where scores are zero;
  32 U sum p |v| for the weights, their sum, the products' second terms and the division;
  a rounding of independent operands to 11 bits is off by 2^-12 of each term at most, uniformly: a sum of them by
      6 * 2^-12 / sqrt(3) * sqrt(sum of squares) in no one of a million cases. Few rows in 16 bits round p s (terms p s e);
      prompts in 16 bits round p and v (two such terms of p v), f16 only v;
  f16 has no step below 2^-24: a weight is off by half of it relative to the factor that f16 weights carry (`floor`);
  the tensor cores' accumulators truncate: each product of 16 slots takes up to 2^-24 of the sum so far, which is at most the
      output and six of its spreads, taken twice for the alignment of the products themselves. For 16-bit prompts that is all the
      tiles of an item (four products each, eight for f16), for few rows in 16 bits the units of a warp;
  half a step of the output type, 2^-8 (bf16), 2^-11 (f16; below 2^-14 f16's steps are 2^-24), 2^-24 (f32) of the value."""
import math

import numpy as np
import pytest

import swiftlet_b200 as swl
from test_gpu_kv4 import NAMES, U, Cache, _torch, quantise

pytestmark = pytest.mark.gpu
HALF = [2.0 ** -24, 2.0 ** -8, 2.0 ** -11]
SIX = 6 / math.sqrt(3)


def put(c, k, v, lens, dtype):
    """Appends k and v (f32 tensors [rows][kvh][hd] on the CPU) as whole sequences; returns what the cache holds, in 64 bits."""
    torch, dts = _torch()
    x = torch.stack([k, v]).to(dts[dtype])
    d = x.cuda()
    swl.kv4_append_device(c.desc(), c.batch(lens, lens), d[0].data_ptr(), d[1].data_ptr(), dtype=dtype)
    torch.cuda.synchronize()
    return torch.from_numpy(quantise(x.float().numpy(), c.group)).cuda().double()


def call(c, lens, new, q, scale, dtype, weights=None, gate=None, want_lse=True):
    """q [rows][heads][hd] of the type; returns out and lse in 64 bits."""
    torch, _ = _torch()
    H, hd = q.shape[1:]
    b = c.batch(lens, new)
    nb = swl.kv4_attention_workspace(c.desc(), b, H)
    work = torch.full((nb,), 255, dtype=torch.uint8, device="cuda")
    out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device="cuda")
    swl.kv4_attention_device(c.desc(), b, H, q.data_ptr(), out.data_ptr(), scale=scale, dtype=dtype,
                             d_gate=0 if gate is None else gate.data_ptr(), d_lse=lse.data_ptr() if want_lse else 0,
                             d_weights=0 if weights is None else weights.data_ptr(),
                             weights_stride=0 if weights is None else weights.stride(1), d_work=work.data_ptr(), work_bytes=nb)
    torch.cuda.synchronize()
    assert int(c.status) == 0
    return out, lse


def exact(k, v, q, scale, n, group):
    """One sequence in 64 bits: k, v [slots][kvh][hd], q [n][heads][hd], the last n slots the rows' own. Per row and head the output,
    lse, the largest sum |q k| scale, sum p |v|, sqrt(sum (p v)^2) and sqrt(sum (p s e)^2) (s e at most: half the group's range)."""
    torch, _ = _torch()
    m, kvh, hd = k.shape
    H = q.shape[1]
    rep = H // kvh
    g = v.view(m, kvh, hd // group, group)
    half = ((g.amax(-1) - g.amin(-1)) / 2).repeat_interleave(group, -1)
    res = [[] for _ in range(6)]
    seen = torch.arange(m, device="cuda")[None] <= (m - n + torch.arange(n, device="cuda"))[:, None]
    for h in range(H):
        kh, vh, sh, qh = k[:, h // rep], v[:, h // rep], half[:, h // rep], q[:, h].double()
        x = (scale * (qh @ kh.T)).masked_fill(~seen, -math.inf)
        z = x.logsumexp(1)
        p = (x - z[:, None]).exp()
        mag = (abs(scale) * (qh.abs() @ kh.abs().T)).masked_fill(~seen, 0).amax(1)
        for r, t in zip(res, (p @ vh, z, mag, p @ vh.abs(), ((p * p) @ (vh * vh)).sqrt(), ((p * p) @ (sh * sh)).sqrt())):
            r.append(t)
    return [torch.stack(r, 1) for r in res]


def bound(e, dtype, few, floor, slots, ds=None):
    """What an output may be off by; e: of `exact`, floor: step of a weight times the sum of what it multiplies."""
    want, _, mag, pabs, pv, pse = e
    ds = (16 * U * mag if ds is None else ds)[..., None]
    tol = (HALF[dtype] * want.abs()).clamp(min=2.0 ** -25 if dtype == 2 else 0) + (2 * ds + 32 * U) * pabs + floor
    if dtype:
        tol = tol + SIX * 2.0 ** -12 * (pse if few else pv * (math.sqrt(2) if dtype == 1 else 1))
        products = slots / 16 / 12 + 1 if few else slots / 16 * dtype
        tol = tol + 2 * products * U * (want.abs() + 6 * (pse if few else pv))
    return tol


def lse_bound(e, ds=None):
    return (16 * U * e[2] if ds is None else ds) + 8 * U * (1 + e[1].abs())


@pytest.mark.parametrize("dtype", [0, 1, 2], ids=NAMES)
@pytest.mark.parametrize("lens,new,kvh,rep,hd,group", [([9000], [1], 2, 8, 256, 64), ([6000, 31, 2500], [1, 3, 4], 2, 8, 256, 128),
                                                       ([5000, 700], [1, 2], 8, 4, 128, 128), ([4100], [150], 2, 8, 256, 64),
                                                       ([700, 3300], [300, 33], 4, 4, 128, 64), ([2900], [200], 1, 8, 64, 64)])
def test_outputs_relative_to_what_is_summed(lens, new, kvh, rep, hd, group, dtype):
    torch, dts = _torch()
    gen = torch.Generator().manual_seed(sum(lens) + hd)
    c = Cache(len(lens), max(lens), kvh, hd, group)
    held = put(c, *(torch.randn(sum(lens), kvh, hd, generator=gen) for _ in range(2)), lens, dtype)
    q = torch.randn(sum(new), kvh * rep, hd, generator=gen).to(dts[dtype]).cuda()
    scale = 1 / math.sqrt(hd)
    out, lse = call(c, lens, new, q, scale, dtype)
    few = max(new) * rep <= 64
    j = s = 0
    for m, n in zip(lens, new):
        e = exact(held[0, s:s + m], held[1, s:s + m], q[j:j + n], scale, n, group)
        err = (out[j:j + n].double() - e[0]).abs()
        tol = bound(e, dtype, few, 0.0, m)
        assert (err <= tol).all(), float((err / tol).max())
        assert ((lse[j:j + n].double() - e[1]).abs() <= lse_bound(e)).all()
        j, s = j + n, s + m


# -------------------------------------------------- keys far from zero, lse --
@pytest.mark.parametrize("dtype", [1, 2], ids=NAMES[1:])
@pytest.mark.parametrize("hd,group", [(256, 64), (256, 128), (128, 64), (128, 128), (64, 64)])
def test_prompts_of_16_bits_without_weights_are_those_with_them(hd, group, dtype):
    """Outputs and lse do not depend on whether weights are accumulated, and lse is an f32 result whatever the inputs' type: keys two
    spreads from zero, which have large common terms, are no less exact."""
    torch, dts = _torch()
    n, slots, kvh, rep = 100, 900, 2, 8
    gen = torch.Generator().manual_seed(hd + group)
    c = Cache(1, slots, kvh, hd, group)
    held = put(c, torch.randn(slots, kvh, hd, generator=gen) + 2, torch.randn(slots, kvh, hd, generator=gen), [slots], dtype)
    q = torch.randn(n, kvh * rep, hd, generator=gen).to(dts[dtype]).cuda()
    scale = 1 / math.sqrt(hd)
    w = torch.zeros(1, kvh, slots, device="cuda")
    out, lse = call(c, [slots], [n], q, scale, dtype)
    out_w, lse_w = call(c, [slots], [n], q, scale, dtype, weights=w)
    out_n, _ = call(c, [slots], [n], q, scale, dtype, want_lse=False)
    e = exact(held[0], held[1], q, scale, n, group)
    assert ((lse.double() - e[1]).abs() <= lse_bound(e)).all(), float((lse.double() - e[1]).abs().max())
    tol = bound(e, dtype, False, 0.0, slots)
    assert ((out.double() - e[0]).abs() <= tol).all()
    assert torch.equal(lse, lse_w) and torch.equal(out, out_w) and torch.equal(out, out_n)


# ------------------------------------------------------------ peaked rows --
def sink(slots, n, ahead, dtype, hd=128, kvh=2, rep=4, seed=0):
    """Queries that slot 0's key puts `ahead` nats before the logarithm of all the others' mean, its value zero; the others' values
    about 0.7: outputs are sums of many small weights."""
    torch, dts = _torch()
    gen = torch.Generator().manual_seed(seed)
    c = Cache(1, slots, kvh, hd)
    k = torch.randn(slots, kvh, hd, generator=gen) * 0.7
    k[0] = torch.randn(kvh, hd, generator=gen).sign() * 2
    v = torch.rand(slots, kvh, hd, generator=gen) + 0.2
    v[0] = 0
    held = put(c, k, v, [slots], dtype)
    scale = 1 / math.sqrt(hd)
    q = torch.randn(n, kvh * rep, hd, generator=gen).cuda().double()
    for h in range(kvh * rep):
        kh = held[0, :, h // rep]
        for _ in range(3):  # the rest moves a little with q's new part
            x = scale * (q[:, h] @ kh.T)
            rest = x[:, 1:].logsumexp(1) - math.log(slots - 1)
            q[:, h] += ((ahead + rest - x[:, 0]) / (scale * (kh[0] @ kh[0])))[:, None] * kh[0]
    q = q.to(dts[dtype])
    return c, held, q, scale


@pytest.mark.parametrize("dtype", [0, 1, 2], ids=NAMES)
@pytest.mark.parametrize("slots", [2000, 30000])
@pytest.mark.parametrize("ahead", [10, 14, 18])
def test_prompts_with_a_dominant_slot(ahead, slots, dtype):
    """f16 weights carry 2^11 (f32 inputs) or 2^7 at the row's reference: half of f16's smallest step is 2^-36 or 2^-32 of it. Steps
    of independent weights, so six spreads of a uniform one."""
    torch, _ = _torch()
    n = 40
    c, held, q, scale = sink(slots, n, ahead, dtype)
    e = exact(held[0], held[1], q, scale, n, c.group)
    out, lse = call(c, [slots], [n], q, scale, dtype)
    assert 0.01 * math.exp(-ahead) * slots < float(e[0].mean()) < slots * math.exp(-ahead)  # the small weights are the output
    floor = SIX * (2.0 ** -32 if dtype else 2.0 ** -36) * held[1].square().sum(0).sqrt().repeat_interleave(4, 0)
    tol = bound(e, dtype, False, floor, slots)
    assert ((out.double() - e[0]).abs() <= tol).all(), float(((out.double() - e[0]).abs() / tol).max())
    assert ((lse.double() - e[1]).abs() <= lse_bound(e)).all()


# ------------------------------------------------------ 16 bits at length --
@pytest.mark.parametrize("dtype", [1, 2], ids=NAMES[1:])
@pytest.mark.parametrize("slots", [8000, 131072])
def test_single_tokens_of_16_bits_at_length(slots, dtype):
    """As many items as blocks, so that a block walks whole contexts; scores of nearly zero, so that all weights count alike. The mean
    error (an accumulator that truncates is off to one side) is held to a hundredth of the outputs' size."""
    torch, dts = _torch()
    nseq, kvh, rep, hd = 75, 2, 8, 128
    gen = torch.Generator().manual_seed(slots)
    c = Cache(1, slots, kvh, hd)
    k, v = (torch.randn(slots, kvh, hd, generator=gen) for _ in range(2))
    held = put(c, k, v, [slots], dtype)
    c.table = c.table.expand(nseq, -1).contiguous()  # all sequences read the same pages
    q = (torch.randn(nseq, kvh * rep, hd, generator=gen) * 1e-3).to(dts[dtype]).cuda()
    out, lse = call(c, [slots] * nseq, [1] * nseq, q, 1 / math.sqrt(hd), dtype)
    e = [torch.cat(x) for x in zip(*(exact(held[0], held[1], q[i:i + 1], 1 / math.sqrt(hd), 1, c.group) for i in range(nseq)))]
    err = out.double() - e[0]
    tol = bound(e, dtype, True, 0.0, slots)
    assert (err.abs() <= tol).all(), float((err.abs() / tol).max())
    assert ((lse.double() - e[1]).abs() <= lse_bound(e)).all()
    # independent errors: their mean over N outputs is their rms / sqrt(N) or so; here a twentieth of one output's rounding
    rms = float(e[0].square().mean().sqrt())
    assert abs(float(err.mean())) <= HALF[dtype] * rms / 20, (float(err.mean()), rms)
    # outputs as near as their own rounding (uniform within half a step, which is HALF of the value at most) and that of p s
    own = HALF[dtype] * rms / math.sqrt(3) + 2.0 ** -12 / math.sqrt(3) * float(e[5].square().mean().sqrt())
    assert float(err.square().mean().sqrt()) <= own, (float(err.square().mean().sqrt()), own)


@pytest.mark.parametrize("dtype", [0, 1, 2], ids=NAMES)
@pytest.mark.parametrize("slots", [2000, 30000])
@pytest.mark.parametrize("ahead", [10, 14, 18])
def test_few_rows_with_a_dominant_slot(ahead, slots, dtype):
    """As many items as blocks, so that one block holds the slot and all that is behind it. The product p s is held with the same
    step, carrying 2^10 and the largest scale's exponent: below 2^-35 of the reference times that scale's binade (scale: range / 15).
    Steps of independent products, so six spreads of a uniform one."""
    torch, _ = _torch()
    n = 75
    c, held, q, scale = sink(slots, n, ahead, dtype, seed=1)
    c.table = c.table.expand(n, -1).contiguous()
    e = [torch.cat(x) for x in zip(*(exact(held[0], held[1], q[i:i + 1], scale, 1, c.group) for i in range(n)))]
    out, lse = call(c, [slots] * n, [1] * n, q, scale, dtype)
    # ranges are below 1 (values 0.2 to 1.2), the largest above 15 / 16: the largest scale is in [2^-4, 2^-3)
    floor = SIX * 2.0 ** -35 * 2.0 ** -4 * 7.5 * math.sqrt(slots)
    tol = bound(e, dtype, True, floor, slots)
    assert ((out.double() - e[0]).abs() <= tol).all(), float(((out.double() - e[0]).abs() / tol).max())
    assert ((lse.double() - e[1]).abs() <= lse_bound(e)).all()


# ------------------------------------------------------------------- gates --
@pytest.mark.parametrize("new", [1, 40])
def test_gates_of_any_size(new):
    """out sigmoid(gate) from -85 (a factor of 1e-37) to 85: the exponential and the quotient are off by 2 units each (CUDA's documented
    bounds for expf and __fdividef), the sum and the product by a rounding."""
    torch, _ = _torch()
    gen = torch.Generator().manual_seed(new)
    c = Cache(1, 150, 2, 128)
    put(c, *(torch.randn(150, 2, 128, generator=gen) for _ in range(2)), [150], 0)
    q = torch.randn(new, 8, 128, generator=gen).cuda()
    gate = torch.linspace(-85, 85, new * 8 * 128).view(new, 8, 128).cuda()
    plain, _ = call(c, [150], [new], q, 0.09, 0)
    gated, _ = call(c, [150], [new], q, 0.09, 0, gate=gate)
    want = plain.double() * gate.double().sigmoid()
    # two units are 4 U
    assert ((gated.double() - want).abs() <= 10 * U * want.abs() + 2.0 ** -149).all()


# ---------------------------------------------------------- large queries --
@pytest.mark.parametrize("dtype", [0, 1], ids=["f32", "bf16"])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("gain", [1e30, 1e-30])
def test_queries_of_any_size(gain, new, dtype):
    """Queries and a scale that undoes them: f32 and bf16 hold both."""
    torch, dts = _torch()
    gen = torch.Generator().manual_seed(new)
    c = Cache(1, 200, 2, 128)
    held = put(c, *(torch.randn(200, 2, 128, generator=gen) for _ in range(2)), [200], dtype)
    q = (torch.randn(new, 8, 128, generator=gen) * gain).to(dts[dtype]).cuda()
    scale = float(np.float32(0.09 / gain))
    w = torch.zeros(1, 2, 200, device="cuda")
    out, lse = call(c, [200], [new], q, scale, dtype, weights=w)
    e = exact(held[0], held[1], q, scale, new, c.group)
    assert ((out.double() - e[0]).abs() <= bound(e, dtype, new == 1, 0.0, 200)).all()
    assert ((lse.double() - e[1]).abs() <= lse_bound(e)).all()
    # every row's weights sum to one, each off by its score's error and that of lse
    assert ((w.double().sum(2) / (4 * new) - 1).abs() <= 2 * 16 * U * e[2].max() + 64 * U).all()


# -------------------------------------------- NaN and lost pages, 16 bits --
@pytest.mark.parametrize("dtype", [1, 2], ids=NAMES[1:])
@pytest.mark.parametrize("new", [1, 5, 40])
def test_what_16_bit_rows_do_not_see(new, dtype):
    """A NaN key and a NaN value in the last slot, a NaN and an infinite query in the last row, a page outside the pool: the rows before
    the last are as exact as without them, the last one is NaN where it has to be."""
    torch, dts = _torch()
    slots, kvh, rep, hd = 300, 2, 8, 256
    gen = torch.Generator().manual_seed(new)
    c = Cache(1, slots, kvh, hd, page=32)
    k, v = (torch.randn(slots, kvh, hd, generator=gen) for _ in range(2))
    k[-1, 0, 3], v[-1, 1, 70] = math.nan, math.inf
    held = put(c, k, v, [slots], dtype)
    q = torch.randn(new, kvh * rep, hd, generator=gen).to(dts[dtype]).cuda()
    q[-1, 9, 0], q[-1, 10, 5] = math.nan, math.inf
    out, lse = call(c, [slots], [new], q, 1 / 16, dtype)
    assert out[-1, :8].isnan().all() and lse[-1, :8].isnan().all() and out[-1, 9:11].isnan().all()
    assert out[-1, 8:, 64:128].isnan().all()
    for h in (8, 11, 15):
        assert out[-1, h, :64].isfinite().all() and out[-1, h, 128:].isfinite().all() and lse[-1, h].isfinite()
    if new > 1:
        e = exact(held[0, :-1], held[1, :-1], q[:-1], 1 / 16, new - 1, c.group)
        assert ((out[:-1].double() - e[0]).abs() <= bound(e, dtype, new * rep <= 64, 0.0, slots)).all()
        assert ((lse[:-1].double() - e[1]).abs() <= lse_bound(e)).all()
    c.table[0, 2] = c.num  # slots 64 .. 95
    b = c.batch([slots - 1], [new])
    q = torch.randn(new, kvh * rep, hd, generator=gen).to(dts[dtype]).cuda()
    nb = swl.kv4_attention_workspace(c.desc(), b, kvh * rep)
    work = torch.full((nb,), 255, dtype=torch.uint8, device="cuda")
    out, lse, w = torch.empty_like(q), torch.empty(new, kvh * rep, device="cuda"), torch.zeros(1, kvh, slots, device="cuda")
    swl.kv4_attention_device(c.desc(), b, kvh * rep, q.data_ptr(), out.data_ptr(), scale=1 / 16, dtype=dtype, d_lse=lse.data_ptr(),
                             d_weights=w.data_ptr(), weights_stride=slots, d_work=work.data_ptr(), work_bytes=nb)
    torch.cuda.synchronize()
    assert int(c.status) == 2 and (w[0, :, 64:96] == 0).all()
    rest = torch.cat([held[:, :64], held[:, 96:-1]], 1)
    e = exact(rest[0], rest[1], q, 1 / 16, new, c.group)
    assert ((out.double() - e[0]).abs() <= bound(e, dtype, new * rep <= 64, 0.0, slots)).all()
    assert ((lse.double() - e[1]).abs() <= lse_bound(e)).all()
    assert ((w.double().sum(2) / (new * rep) - 1).abs() <= 2 * 16 * U * e[2].max() + 64 * U).all()
