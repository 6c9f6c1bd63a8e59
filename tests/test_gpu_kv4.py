"""The 4-bit KV cache operators against plain implementations in 64 bits.

Tolerances. Quantised values and evictions are exact. An attention output is
off by: the score's f32 rounding, at most 16 roundings' worth (the square
root of 256 terms) of sum |q k| scale, which changes a weight by that share
(twice: the weight and the sum); a few roundings of the weights, sums and the
final division (32 units) relative to the largest value; for 16-bit types the
rounding of weights and of dequantised keys and values to 11 bits on their way
into the tensor cores (each half a step, 2^-12; the keys' enters a score with
the square root of the sum of squares, four of them); and half a step of the
output type."""
import math

import numpy as np
import pytest

import swiftlet_b200 as swl

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
NAMES = ["f32", "bf16", "f16"]


def _torch():
    import torch
    return torch, [torch.float32, torch.bfloat16, torch.float16]


def quantise(x, group):
    """Values that x (float32) stands for in the cache."""
    f = np.float32
    y = x.reshape(*x.shape[:-1], -1, group)
    with np.errstate(all="ignore"):
        mn, mx = y.min(-1, keepdims=True), y.max(-1, keepdims=True)
        b, s = mn.astype(np.float16), ((mx - mn) * f(1 / 15)).astype(np.float16)
        bf, sf = b.astype(f), s.astype(f)
        inv = np.where(sf > 0, f(1) / sf, f(0))
        q = np.clip(np.rint((y - bf) * inv), 0, 15)
        v = (q * sf + bf).astype(f)
        bad = ~np.isfinite(y).all(-1, keepdims=True) | ~np.isfinite(bf) | ~np.isfinite(sf)
    return np.where(bad, f(np.nan), v).reshape(x.shape)


class Cache:
    """A pool full of NaN bytes, a scattered page table, and what the slots hold ([2][nseq][slots][kvh][hd])."""

    def __init__(self, nseq, max_len, kvh, hd, group=64, page=64, seed=0, spare=0):
        torch, _ = _torch()
        rng = np.random.default_rng(seed)
        self.kvh, self.hd, self.group, self.page, self.max_len, self.nseq = kvh, hd, group, page, max_len, nseq
        self.per = max(1, -(-max_len // page))
        n = nseq * self.per + spare + 1
        self.pool = torch.full((n * swl.kv4_page_bytes(kvh, hd, group, page),), 255, dtype=torch.uint8, device="cuda")
        order = rng.permutation(n).astype(np.int32)
        self.spare = order[nseq * self.per:]
        self.table = torch.from_numpy(order[:nseq * self.per].reshape(nseq, self.per)).cuda()
        self.num = n
        self.held = np.full((2, nseq, max_len, kvh, hd), np.nan, np.float32)
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def desc(self, table=None):
        t = self.table if table is None else table
        return swl.swl_kv4_cache(self.pool.data_ptr(), t.data_ptr(), t.stride(0), self.num, self.page, self.kvh, self.hd, self.group)

    def batch(self, lens, new, max_len=None):
        torch, _ = _torch()
        start = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device="cuda")
        dl = torch.tensor(np.asarray(lens), dtype=torch.int32, device="cuda")
        b = swl.swl_kv4_batch(start.data_ptr(), dl.data_ptr(), len(lens), int(sum(new)), int(max(list(new) + [0])),
                              self.max_len if max_len is None else max_len, self.status.data_ptr())
        b.keep = (start, dl)
        return b

    def append(self, lens, new, rng, dtype=0, scale=1.0):
        torch, dts = _torch()
        rows = sum(new)
        x = torch.from_numpy((rng.standard_normal((2, max(rows, 1), self.kvh, self.hd)) * scale).astype(np.float32)).to(dts[dtype])
        d = x.cuda()
        swl.kv4_append_device(self.desc(), self.batch(lens, new), d[0].data_ptr(), d[1].data_ptr(), dtype=dtype)
        torch.cuda.synchronize()
        v = quantise(x.float().numpy(), self.group)
        j = 0
        for i, (m, n) in enumerate(zip(lens, new)):
            for t in range(n):
                if m - n + t >= 0:
                    self.held[:, i, m - n + t] = v[:, j]
                j += 1

    def fill(self, lens, rng, dtype=0):
        self.append(lens, lens, rng, dtype)


def attend(c, lens, new, rep, rng, dtype=0, scale=None, gate=False, weights=None, table=None, stream=0, qgain=1.2):
    """Runs the call; returns (out, lse, weights) as float64 numpy and the inputs."""
    torch, dts = _torch()
    H, rows, hd = c.kvh * rep, sum(new), c.hd
    scale = 1 / math.sqrt(hd) if scale is None else scale
    # q and gate interleaved per head, as the model's projection lays them out
    qg = torch.from_numpy((rng.standard_normal((rows, H, 2, hd)) * qgain).astype(np.float32)).to(dts[dtype]).cuda()
    out = torch.full((rows + 2, H, hd), 7.0, dtype=dts[dtype], device="cuda")
    lse = torch.full((rows + 2, H), 7.0, device="cuda")
    b = c.batch(lens, new)
    nb = swl.kv4_attention_workspace(c.desc(table), b, H)
    work = torch.full((nb,), 255, dtype=torch.uint8, device="cuda")
    e = qg.element_size()
    swl.kv4_attention_device(c.desc(table), b, H, qg.data_ptr(), out.data_ptr(), scale=scale, dtype=dtype,
                             q_strides=(2 * H * hd, 2 * hd), d_gate=qg.data_ptr() + hd * e if gate else 0,
                             gate_strides=(2 * H * hd, 2 * hd), d_lse=lse.data_ptr(),
                             d_weights=0 if weights is None else weights.data_ptr(),
                             weights_stride=0 if weights is None else weights.stride(1), d_work=work.data_ptr(), work_bytes=nb)
    torch.cuda.synchronize()
    assert (out[rows:].float() == 7).all() and (lse[rows:] == 7).all()  # rows behind the last sequence
    q = qg.float().cpu().numpy().astype(np.float64)
    return out[:rows].float().cpu().numpy().astype(np.float64), lse[:rows].cpu().numpy().astype(np.float64), q


def check(c, lens, new, rep, got, lse, q, dtype=0, scale=None, gate=False, weights=None, before=None, held=None):
    scale = 1 / math.sqrt(c.hd) if scale is None else scale
    held = c.held if held is None else held
    half = {0: 2.0 ** -24, 1: 2.0 ** -8 / 2, 2: 2.0 ** -11 / 2}[dtype] * 1.01
    narrow = 2.0 ** -12 if dtype else 0.0
    j = 0
    for i, (m, n) in enumerate(zip(lens, new)):
        wsum = np.zeros((c.kvh, max(m, 1)))
        wtol = 0.0
        for t in range(n):
            seen = max(0, min(m, m - n + t + 1))
            for h in range(c.kvh * rep):
                if seen == 0:
                    assert (got[j, h] == 0).all() and lse[j, h] == -np.inf
                    continue
                k, v = (held[w, i, :seen, h // rep].astype(np.float64) for w in (0, 1))
                x = scale * (k @ q[j, h, 0])
                z = x.max() + np.log(np.exp(x - x.max()).sum())
                p = np.exp(x - z)
                mag = np.abs(k) @ np.abs(q[j, h, 0]) * abs(scale)
                sq = np.sqrt((k * k) @ (q[j, h, 0] ** 2)) * abs(scale)
                ds = (16 * U * mag + 4 * narrow * sq).max()  # of a score
                want = p @ v
                vmax = np.abs(v).max()
                tol = (2 * ds + 32 * U + 2 * narrow) * vmax
                if gate:
                    g = 1 / (1 + np.exp(-q[j, h, 1]))
                    want, tol = want * g, tol + 4 * U * vmax
                err = np.abs(got[j, h] - want) - half * np.abs(want)
                assert err.max() <= tol, (i, t, h, err.max(), tol)
                assert abs(lse[j, h] - z) <= ds + 8 * U * (1 + abs(z)) + narrow, (i, t, h, lse[j, h], z)
                wsum[h // rep, :seen] += p
                wtol = max(wtol, 2 * ds + 32 * U)
            j += 1
        if weights is not None:
            w0, w1 = before[i, :, :m], weights[i, :, :m]
            # an f32 sum is off by its roundings relative to the terms' sizes, |w0| + sum (w0 may be negative: the sum of the two is then
            # below either, and no bound on the error)
            assert (np.abs(w1 - (w0 + wsum[:, :m])) <= wtol * (wsum[:, :m] + 1e-30) + 8 * U * (np.abs(w0) + wsum[:, :m])).all(), i
            assert (weights[i, :, m:] == before[i, :, m:]).all()


# ------------------------------------------------------------ append, read --
@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("kvh,hd,group,page", [(2, 256, 64, 64), (1, 64, 64, 16), (3, 128, 128, 32), (2, 128, 64, 128), (5, 256, 128, 16)])
def test_append_and_read_are_exact(kvh, hd, group, page, dtype):
    torch, dts = _torch()
    rng = np.random.default_rng(hd + page + dtype)
    c = Cache(5, 150, kvh, hd, group, page)
    lens, new = [1, 150, 0, 77, 16], [1, 150, 0, 3, 16]
    c.held[:] = 0
    c.append([0, 0, 0, 74, 0], [0, 0, 0, 74, 0], rng, dtype)
    c.append(lens, new, rng, dtype)
    # strided and oddly aligned destinations
    rows = sum(new)
    back = torch.full((2, rows + 1, kvh, hd + 3), 7.0, dtype=dts[dtype], device="cuda")
    st = (kvh * (hd + 3), hd + 3)
    swl.kv4_read_device(c.desc(), c.batch(lens, new), back[0, :, :, 1:].data_ptr(), back[1].data_ptr(), dtype=dtype, k_strides=st,
                        v_strides=st)
    torch.cuda.synchronize()
    assert (back[:, rows:] == 7).all() and (back[0, :, :, 0] == 7).all() and (back[1, :, :, hd:] == 7).all()
    got = [back[0, :rows, :, 1:hd + 1].cpu(), back[1, :rows, :, :hd].cpu()]
    want = np.concatenate([c.held[:, i, m - n:m] for i, (m, n) in enumerate(zip(lens, new))], axis=1)
    for w in (0, 1):
        assert torch.equal(got[w], torch.from_numpy(want[w]).to(dts[dtype]))
    assert int(c.status) == 0


def test_quantisation_error_is_half_a_step():
    rng = np.random.default_rng(3)
    c = Cache(1, 300, 2, 256)
    x = rng.standard_normal((300, 2, 256)).astype(np.float32)
    y = x.reshape(300, 2, 4, 64)
    step = (y.max(-1) - y.min(-1)) / 15
    err = np.abs(quantise(x, 64).reshape(y.shape) - y).max(-1)
    # half a step, the roundings of bias (|b| 2^-11) and of 15 scales (2^-11 each)
    assert (err <= step * (0.5 + 15 * 2.0 ** -11) + np.abs(y.min(-1)) * 2.0 ** -11).all()


def test_append_of_odd_values():
    """Constant groups, tiny and huge ranges, NaN, infinities and values beyond f16; more tokens than slots."""
    torch, _ = _torch()
    c = Cache(1, 40, 1, 64)
    x = np.random.default_rng(0).standard_normal((12, 1, 64)).astype(np.float32)
    x[0], x[1], x[2] = 0.0, 3.25, x[2] * 1e-9
    x[3], x[4, 0, 5], x[5, 0, 6] = x[3] * 2e4, np.nan, np.inf
    x[6, 0, 0], x[7, 0, 1] = 7e4, -np.inf
    x[8, 0, :32] = -0.0
    x[9] *= 60000 / np.abs(x[9]).max()
    d = torch.from_numpy(x).cuda()
    back = torch.zeros_like(d)
    back2 = torch.zeros_like(d)
    swl.kv4_append_device(c.desc(), c.batch([12], [12]), d.data_ptr(), d.data_ptr())
    swl.kv4_read_device(c.desc(), c.batch([12], [12]), back.data_ptr(), back2.data_ptr())
    torch.cuda.synchronize()
    want = quantise(x, 64)
    for b in (back, back2):
        assert np.array_equal(b.cpu().numpy(), want, equal_nan=True)
    assert np.isnan(want[[4, 5, 7]]).all() and not np.isnan(want[[0, 1, 2, 3, 8, 9]]).any() and (want[1] == 3.25).all()
    # five slots for twelve tokens: the last five are kept
    swl.kv4_append_device(c.desc(), c.batch([5], [12]), d.data_ptr(), d.data_ptr())
    back.fill_(7)
    swl.kv4_read_device(c.desc(), c.batch([5], [5]), back.data_ptr(), back2.data_ptr())
    torch.cuda.synchronize()
    assert np.array_equal(back[:5].cpu().numpy(), want[7:], equal_nan=True)


def test_append_clears_the_weights_of_new_slots():
    torch, _ = _torch()
    c = Cache(2, 70, 2, 128)
    w = torch.full((2, 2, 75), 3.0, device="cuda")
    x = torch.randn(8, 2, 128, device="cuda")
    swl.kv4_append_device(c.desc(), c.batch([66, 5], [3, 5]), x.data_ptr(), x.data_ptr(), d_weights=w.data_ptr(), weights_stride=75)
    want = torch.full_like(w, 3.0)
    want[0, :, 63:66] = 0
    want[1, :, :5] = 0
    torch.cuda.synchronize()
    assert torch.equal(w, want)


# ---------------------------------------------------------------- attention --
SHAPES = [(2, 8, 256, 64, 64), (1, 8, 256, 128, 16), (2, 2, 128, 64, 32), (4, 4, 128, 128, 16), (8, 1, 64, 64, 64), (1, 8, 64, 64, 128),
          (2, 6, 128, 64, 64), (1, 16, 128, 64, 128), (1, 3, 256, 64, 32), (1, 64, 64, 64, 64), (3, 5, 64, 64, 16)]


@pytest.mark.parametrize("dtype", [0, 1, 2], ids=NAMES)
@pytest.mark.parametrize("kvh,rep,hd,group,page", SHAPES)
def test_single_tokens(kvh, rep, hd, group, page, dtype):
    rng = np.random.default_rng(hd + rep + page)
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 0, 515]
    c = Cache(len(lens), 515, kvh, hd, group, page, seed=rep)
    c.fill(lens, rng, dtype)
    new = [1] * len(lens)
    got, lse, q = attend(c, lens, new, rep, rng, dtype, gate=True)
    check(c, lens, new, rep, got, lse, q, dtype, gate=True)
    assert int(c.status) == 0


@pytest.mark.parametrize("dtype", [0, 1, 2], ids=NAMES)
@pytest.mark.parametrize("kvh,rep,hd,group,page", SHAPES)
def test_prompts(kvh, rep, hd, group, page, dtype):
    rng = np.random.default_rng(hd * rep + page)
    lens = [40, 1, 200, 0, 130, 64, 9]
    new = [40, 1, 17, 0, 1, 64, 12]  # the last has more tokens than slots
    c = Cache(len(lens), 200, kvh, hd, group, page, seed=rep)
    c.fill([max(0, m - n) for m, n in zip(lens, new)], rng, dtype)
    c.append(lens, new, rng, dtype)
    got, lse, q = attend(c, lens, new, rep, rng, dtype)
    check(c, lens, new, rep, got, lse, q, dtype)
    assert int(c.status) == 0


@pytest.mark.parametrize("dtype", [0, 1], ids=["f32", "bf16"])
@pytest.mark.parametrize("lens,new", [([9000], [1]), ([6000, 3, 2500], [1, 1, 1]), ([2100], [150]), ([700, 1300], [300, 5])])
def test_longer(lens, new, dtype):
    """Contexts that are split over many blocks, and prompts of several tiles, at the head shape of the 35B configuration."""
    rng = np.random.default_rng(sum(lens))
    c = Cache(len(lens), max(lens), 2, 256)
    c.fill(lens, rng, dtype)
    got, lse, q = attend(c, lens, new, 8, rng, dtype, gate=True)
    check(c, lens, new, 8, got, lse, q, dtype, gate=True)


@pytest.mark.parametrize("dtype", [0, 1, 2], ids=NAMES)
@pytest.mark.parametrize("kvh,rep,hd,new", [(2, 8, 256, [1, 1, 1]), (2, 2, 128, [1, 40, 0]), (1, 16, 64, [1, 2, 3]), (2, 6, 128, [70, 1, 1])])
def test_weights_accumulate(kvh, rep, hd, new, dtype):
    torch, _ = _torch()
    rng = np.random.default_rng(hd)
    lens = [200, 137, 90]
    c = Cache(3, 200, kvh, hd)
    c.fill(lens, rng, dtype)
    w = torch.rand(3, kvh, 211, device="cuda")
    before = w.cpu().numpy().astype(np.float64)
    got, lse, q = attend(c, lens, new, rep, rng, dtype, weights=w)
    check(c, lens, new, rep, got, lse, q, dtype, weights=w.cpu().numpy().astype(np.float64), before=before)
    # the sums are the same bits each time
    w1 = torch.zeros_like(w)
    w2 = torch.zeros_like(w)
    attend(c, lens, new, rep, np.random.default_rng(1), dtype, weights=w1)
    attend(c, lens, new, rep, np.random.default_rng(1), dtype, weights=w2)
    assert torch.equal(w1, w2)


@pytest.mark.parametrize("dtype,hd", [(1, 256), (2, 128), (0, 64)])
def test_weights_of_prompts_keep_their_bits(dtype, hd):
    """The weights of a prompt are f32 sums: with keys far from zero they are held to the f32 bound (16 roundings of sum |q k| scale, and
    2^-22 of it for two f16 terms of a key) whatever the inputs' type."""
    torch, dts = _torch()
    rng = np.random.default_rng(21)
    n, new, rep = 600, 100, 8
    c = Cache(1, n, 2, hd)
    x = torch.from_numpy((rng.standard_normal((2, n, 2, hd)) + 2).astype(np.float32)).to(dts[dtype])
    d = x.cuda()
    swl.kv4_append_device(c.desc(), c.batch([n], [n]), d[0].data_ptr(), d[1].data_ptr(), dtype=dtype)
    held = quantise(x.float().numpy(), 64).astype(np.float64)
    w = torch.zeros(1, 2, n, device="cuda")
    _, lse, q = attend(c, [n], [new], rep, rng, dtype=dtype, weights=w)
    want, ds, scale = np.zeros((2, n)), 0.0, 1 / math.sqrt(hd)
    for t in range(new):
        for h in range(2 * rep):
            k = held[0, :n - new + t + 1, h // rep]
            s = scale * (k @ q[t, h, 0])
            z = s.max() + np.log(np.exp(s - s.max()).sum())
            own = (20 * U * scale * (np.abs(k) @ np.abs(q[t, h, 0]))).max()
            assert abs(lse[t, h] - z) <= own + 8 * U * (1 + abs(z))
            ds = max(ds, own)
            want[h // rep, :k.shape[0]] += np.exp(s - z)
    assert (np.abs(w[0].cpu().numpy() - want) <= (2 * ds + 64 * U) * want + 1e-12).all()


def test_values_of_very_different_size():
    """Values from 1e-5 to 1e4 in neighbouring groups and slots, and large scores: nothing under- or overflows on the way."""
    torch, _ = _torch()
    rng = np.random.default_rng(8)
    for gain, qgain in ((1e-4, 1.0), (2e3, 1.0), (1.0, 60.0)):
        c = Cache(1, 400, 2, 256)
        c.append([400], [400], rng, 0, scale=gain)
        got, lse, q = attend(c, [400], [1], 8, rng, 0, scale=1 / (16 * gain), qgain=qgain)
        check(c, [400], [1], 8, got, lse, q, 0, scale=1 / (16 * gain))
    c = Cache(1, 400, 2, 256)
    x = rng.standard_normal((2, 400, 2, 256)).astype(np.float32)
    x[1] *= np.exp(rng.uniform(-9, 9, (400, 2, 4))).repeat(64, -1).astype(np.float32)
    d = torch.from_numpy(x).cuda()
    swl.kv4_append_device(c.desc(), c.batch([400], [400]), d[0].data_ptr(), d[1].data_ptr())
    c.held[:, 0] = quantise(x, 64)
    for new in ([1], [30]):
        got, lse, q = attend(c, [400], new, 8, rng)
        check(c, [400], new, 8, got, lse, q)


def test_nan_and_infinity_stay_where_they_are():
    """A NaN key or value that a row does not see changes nothing; one that it sees makes that row (value: that group) NaN; a NaN
    query makes its own row NaN."""
    torch, _ = _torch()
    rng = np.random.default_rng(2)
    for new in (1, 6, 40):
        c = Cache(2, 150, 2, 256)
        x = rng.standard_normal((2, 300, 2, 256)).astype(np.float32)
        x[0, 149, 0, 3] = np.nan   # last key of sequence 0, head 0
        x[1, 299, 1, 70] = np.inf  # last value of sequence 1, head 1, group 1
        d = torch.from_numpy(x).cuda()
        swl.kv4_append_device(c.desc(), c.batch([150, 150], [150, 150]), d[0].data_ptr(), d[1].data_ptr())
        c.held[:] = quantise(x, 64).reshape(2, 2, 150, 2, 256)
        got, lse, q = attend(c, [150, 150], [new, new], 8, rng)
        a, b = new - 1, 2 * new - 1
        assert np.isnan(got[a, :8]).all() and np.isnan(lse[a, :8]).all()
        assert np.isnan(got[b, 8:, 64:128]).all()
        ok = np.ones_like(got, bool)
        ok[a, :8] = False
        ok[b, 8:, 64:128] = False
        assert np.isfinite(got[ok]).all()
        seen = np.where(np.isnan(c.held), 0, c.held)
        sub = [i for i in range(2 * new) if i not in (a, b)]
        if sub:
            lens2, new2 = [149, 149], [new - 1, new - 1]
            check(c, lens2, new2, 8, got[sub], lse[sub], q[sub], held=seen)


@pytest.mark.parametrize("dtype", [0, 1], ids=["f32", "bf16"])
def test_nan_value_leaves_other_rows_their_bits(dtype):
    """A value group that reads as NaN, in the last of a few new tokens: the rows before it do not see it, and are as exact as
    without it (queries so small that a score's own error is no part of the bound)."""
    torch, _ = _torch()
    rng = np.random.default_rng(8)
    c = Cache(1, 20, 2, 256)
    x = rng.standard_normal((2, 20, 2, 256)).astype(np.float32)
    x[1, 19, :, 70] = np.inf
    d = torch.from_numpy(x).cuda()
    swl.kv4_append_device(c.desc(), c.batch([20], [20]), d[0].data_ptr(), d[1].data_ptr())
    c.held[:] = quantise(x, 64).reshape(2, 1, 20, 2, 256)
    got, lse, q = attend(c, [20], [2], 8, rng, dtype=dtype, qgain=0.02)
    assert np.isnan(got[1, :, 64:128]).all()
    check(c, [19], [1], 8, got[:1], lse[:1], q[:1], dtype=dtype, held=c.held)


def test_nan_query_stays_in_its_row():
    torch, _ = _torch()
    for new in (1, 20):
        c = Cache(1, 100, 1, 128)
        c.fill([100], np.random.default_rng(0))
        q = torch.randn(new, 8, 128, device="cuda")
        out0, out1 = torch.empty_like(q), torch.empty_like(q)
        b = c.batch([100], [new])
        n = swl.kv4_attention_workspace(c.desc(), b, 8)
        work = torch.empty(n, dtype=torch.uint8, device="cuda")
        swl.kv4_attention_device(c.desc(), b, 8, q.data_ptr(), out0.data_ptr(), scale=0.1, d_work=work.data_ptr(), work_bytes=n)
        q[new - 1, 3, 7] = float("nan")
        q[new - 1, 5, 0] = float("inf")
        swl.kv4_attention_device(c.desc(), b, 8, q.data_ptr(), out1.data_ptr(), scale=0.1, d_work=work.data_ptr(), work_bytes=n)
        torch.cuda.synchronize()
        assert torch.isnan(out1[new - 1, [3, 5]]).all()
        out1[new - 1, [3, 5]] = out0[new - 1, [3, 5]]
        assert torch.equal(out0, out1)


def test_bad_pages_and_lengths_are_reported():
    """A page id outside the pool: its slots count as masked. A length outside [0, max_len]: held to it. Both set status bit 1."""
    torch, _ = _torch()
    rng = np.random.default_rng(4)
    for new in (1, 30):
        c = Cache(2, 300, 2, 128, page=32)
        c.fill([300, 300], rng)
        good = c.table.clone()
        for bad in (-1, c.num, 2 ** 31 - 1):
            c.table.copy_(good)
            c.table[0, 2] = bad  # slots 64 .. 95
            c.status.zero_()
            w = torch.zeros(2, 2, 300, device="cuda")
            got, lse, q = attend(c, [300, 300], [new, new], 4, rng, weights=w)
            assert int(c.status) == 2
            assert (w[0, :, 64:96] == 0).all() and np.isfinite(got).all()
            held = np.concatenate([c.held[:, :, :64], c.held[:, :, 96:]], axis=2)
            check(c, [268], [new], 4, got[:new], lse[:new], q[:new], held=held[:, :1])
            check(c, [300], [new], 4, got[new:], lse[new:], q[new:], held=c.held[:, 1:])
            x = torch.zeros(300, 2, 128, device="cuda")
            swl.kv4_read_device(c.desc(), c.batch([300], [300]), x.data_ptr(), torch.empty_like(x).data_ptr())
            torch.cuda.synchronize()
            assert (x[64:96] == 0).all() and (x[96:].cpu().numpy() == c.held[0, 0, 96:]).all()
        c.table.copy_(good)
        for m, as_if in ((301, 300), (2 ** 31 - 1, 300), (-5, 0)):
            c.status.zero_()
            got, lse, q = attend(c, [m, 300], [new, new], 4, rng)
            assert int(c.status) == 2
            check(c, [as_if, 300], [new, new], 4, got, lse, q)


def test_no_lse_and_dense_rows():
    """Without lse, gate and weights; the same bits as with them."""
    torch, _ = _torch()
    for new in ([1, 1], [20, 7]):
        c = Cache(2, 90, 2, 128)
        c.fill([90, 33], np.random.default_rng(0))
        q = torch.randn(sum(new), 4, 128, device="cuda")
        a, b2 = torch.empty_like(q), torch.empty_like(q)
        lse, w = torch.empty(sum(new), 4, device="cuda"), torch.zeros(2, 2, 90, device="cuda")
        b = c.batch([90, 33], new)
        n = swl.kv4_attention_workspace(c.desc(), b, 4)
        work = torch.empty(n, dtype=torch.uint8, device="cuda")
        k = dict(scale=0.09, d_work=work.data_ptr(), work_bytes=n)
        swl.kv4_attention_device(c.desc(), b, 4, q.data_ptr(), a.data_ptr(), **k)
        swl.kv4_attention_device(c.desc(), b, 4, q.data_ptr(), b2.data_ptr(), d_lse=lse.data_ptr(), d_weights=w.data_ptr(),
                                 weights_stride=90, **k)
        w1 = w.clone().zero_()
        swl.kv4_attention_device(c.desc(), b, 4, q.data_ptr(), a.data_ptr(), d_weights=w1.data_ptr(), weights_stride=90, **k)
        torch.cuda.synchronize()
        assert torch.equal(a, b2) and torch.equal(w, w1)


def test_captured_and_replayed_with_other_lengths():
    """A captured graph reads lengths, starts and table when it is replayed; on a stream of its own."""
    torch, _ = _torch()
    rng = np.random.default_rng(6)
    c = Cache(3, 700, 2, 256, spare=2)
    lens = [700, 300, 1]
    c.fill(lens, rng)
    q = torch.randn(3, 16, 256, device="cuda")
    out, lse, w = torch.empty_like(q), torch.empty(3, 16, device="cuda"), torch.zeros(3, 2, 700, device="cuda")
    b = c.batch(lens, [1, 1, 1])
    n = swl.kv4_attention_workspace(c.desc(), b, 16)
    work = torch.empty(n, dtype=torch.uint8, device="cuda")
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        swl.kv4_attention_device(c.desc(), b, 16, q.data_ptr(), out.data_ptr(), scale=1 / 16, d_lse=lse.data_ptr(),
                                 d_weights=w.data_ptr(), weights_stride=700, d_work=work.data_ptr(), work_bytes=n,
                                 stream=torch.cuda.current_stream().cuda_stream)
    for m in (lens, [5, 299, 0], [600, 200, 1]):
        b.keep[1].copy_(torch.tensor(m, dtype=torch.int32))
        w.zero_()
        g.replay()
        torch.cuda.synchronize()
        qq = q.cpu().numpy().astype(np.float64)[:, :, None]
        check(c, m, [1, 1, 1], 8, out.cpu().numpy().astype(np.float64), lse.cpu().numpy().astype(np.float64), qq,
              weights=w.cpu().numpy().astype(np.float64), before=np.zeros((3, 2, 700)))


def test_many_short_sequences():
    """More sequences than a warp has lanes, most of them without new tokens, rows of the buffers left over."""
    rng = np.random.default_rng(12)
    lens = [int(x) for x in rng.integers(0, 40, 150)]
    for new in ([1] * 150, [int(x) for x in rng.integers(0, 4, 150)], [0] * 149 + [30]):
        lens2 = [max(m, n) if n > 4 else m for m, n in zip(lens, new)]
        c = Cache(150, 40, 1, 64, page=16)
        c.fill(lens2, rng)
        got, lse, q = attend(c, lens2, new, 8, rng)
        check(c, lens2, new, 8, got, lse, q)


def test_total_above_the_rows():
    """`total` is a bound: rows between start[nseq] and it belong to nobody and stay as they are."""
    torch, _ = _torch()
    c = Cache(2, 60, 2, 64)
    c.fill([60, 20], np.random.default_rng(0))
    for new in ([1, 1], [9, 20]):
        rows = sum(new)
        b = c.batch([60, 20], new)
        b.total = rows + 40
        q = torch.randn(rows + 40, 16, 64, device="cuda")
        out, lse = torch.full_like(q, 7.0), torch.full((rows + 40, 16), 7.0, device="cuda")
        w = torch.zeros(2, 2, 60, device="cuda")
        n = swl.kv4_attention_workspace(c.desc(), b, 16)
        work = torch.full((n,), 255, dtype=torch.uint8, device="cuda")
        swl.kv4_attention_device(c.desc(), b, 16, q.data_ptr(), out.data_ptr(), scale=0.125, d_lse=lse.data_ptr(), d_weights=w.data_ptr(),
                                 weights_stride=60, d_work=work.data_ptr(), work_bytes=n)
        x, y = torch.full((rows + 40, 2, 64), 7.0, device="cuda"), torch.full((rows + 40, 2, 64), 7.0, device="cuda")
        swl.kv4_read_device(c.desc(), b, x.data_ptr(), y.data_ptr())
        before = c.pool.clone()
        swl.kv4_append_device(c.desc(), b, x.data_ptr(), y.data_ptr())  # what was read, and rows of sevens that have no slot
        swl.kv4_read_device(c.desc(), b, x.data_ptr(), y.data_ptr())
        torch.cuda.synchronize()
        assert (out[rows:] == 7).all() and (lse[rows:] == 7).all() and (x[rows:] == 7).all() and (y[rows:] == 7).all()
        changed = (before != c.pool).view(-1, swl.kv4_page_bytes(2, 64, 64, 64)).any(1).nonzero().flatten().tolist()
        assert set(changed) <= set(c.table.flatten().tolist())
        c.pool.copy_(before)
        check(c, [60, 20], new, 8, out[:rows].cpu().numpy().astype(np.float64), lse[:rows].cpu().numpy().astype(np.float64),
              q[:rows].cpu().numpy().astype(np.float64)[:, :, None], weights=w.cpu().numpy().astype(np.float64), before=np.zeros((2, 2, 60)))


def test_offsets_beyond_32_bits():
    """Pages above 4 GiB of the pool, for every call."""
    torch, _ = _torch()
    rng = np.random.default_rng(5)
    c = Cache(2, 200, 2, 256)
    pb = swl.kv4_page_bytes(2, 256, 64, 64)
    n = (5 << 30) // pb
    c.pool = torch.empty(n * pb, dtype=torch.uint8, device="cuda")
    c.num = n
    c.table = torch.from_numpy((n - 1 - np.arange(8, dtype=np.int32)).reshape(2, 4)).cuda()
    c.spare = n - 9 - np.arange(8, dtype=np.int32)
    c.fill([200, 130], rng)
    for new in ([1, 1], [40, 3]):
        got, lse, q = attend(c, [200, 130], new, 8, rng)
        check(c, [200, 130], new, 8, got, lse, q)
    w = torch.from_numpy(rng.random((2, 2, 200)).astype(np.float32)).cuda()
    check_evict(c, [200, 130], w, 128, 4, 20)


def test_negative_and_zero_scale():
    rng = np.random.default_rng(13)
    for scale in (-0.07, 0.0):
        for new in (1, 20):
            c = Cache(1, 150, 2, 128)
            c.fill([150], rng)
            got, lse, q = attend(c, [150], [new], 4, rng, scale=scale)
            check(c, [150], [new], 4, got, lse, q, scale=scale)


def test_two_calls_at_once():
    """Calls on two streams with workspaces of their own, a captured prompt among them, replayed with other lengths."""
    torch, _ = _torch()
    rng = np.random.default_rng(14)
    c = Cache(3, 900, 2, 256)
    lens = [900, 300, 64]
    c.fill(lens, rng)
    runs = []
    for k, new in enumerate(([1, 1, 1], [70, 5, 20])):
        rows = sum(new)
        q = torch.randn(rows, 16, 256, device="cuda")
        out, lse, w = torch.empty_like(q), torch.empty(rows, 16, device="cuda"), torch.zeros(3, 2, 900, device="cuda")
        b = c.batch(lens, new)
        n = swl.kv4_attention_workspace(c.desc(), b, 16)
        work = torch.empty(n, dtype=torch.uint8, device="cuda")
        s = torch.cuda.Stream()

        def call(stream, q=q, out=out, lse=lse, w=w, b=b, work=work, n=n):
            swl.kv4_attention_device(c.desc(), b, 16, q.data_ptr(), out.data_ptr(), scale=1 / 16, d_lse=lse.data_ptr(),
                                     d_weights=w.data_ptr(), weights_stride=900, d_work=work.data_ptr(), work_bytes=n, stream=stream)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            call(torch.cuda.current_stream().cuda_stream)
        runs.append((new, q, out, lse, w, b, g, s))
    for m in (lens, [500, 5, 63]):
        for new, q, out, lse, w, b, g, s in runs:
            b.keep[1].copy_(torch.tensor(m, dtype=torch.int32))
            w.zero_()
        torch.cuda.synchronize()
        for *_, g, s in runs:
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for new, q, out, lse, w, b, g, s in runs:
            check(c, m, new, 8, out.cpu().numpy().astype(np.float64), lse.cpu().numpy().astype(np.float64),
                  q.cpu().numpy().astype(np.float64)[:, :, None], weights=w.cpu().numpy().astype(np.float64), before=np.zeros((3, 2, 900)))


# -------------------------------------------------------------------- evict --
def survivors(w, n, keep, first, recent):
    if n <= keep:
        return np.arange(n)
    w = np.where(np.isnan(w[:n]), -np.inf, w[:n].astype(np.float64))
    mid = np.arange(first, n - recent)
    top = mid[np.lexsort((mid, -w[mid]))][:keep - first - recent]
    return np.sort(np.concatenate([np.arange(first), top, np.arange(n - recent, n)]))


def run_evict(c, lens, w, keep, first, recent, with_kept=True, with_weights=True):
    torch, _ = _torch()
    most = min(keep, c.max_len)
    per = max(1, -(-most // c.page))
    dst = torch.from_numpy(np.ascontiguousarray(c.spare[:c.nseq * per].reshape(c.nseq, per))).cuda()
    nl = torch.full((c.nseq,), -9, dtype=torch.int32, device="cuda")
    kept = torch.full((c.nseq, c.kvh, most + 2), -9, dtype=torch.int32, device="cuda")
    nw = torch.full((c.nseq, c.kvh, most + 3), -9.0, device="cuda")
    b = c.batch(lens, [0] * c.nseq)
    b.start = None
    nb = swl.kv4_evict_workspace(c.desc(), b, keep)
    work = torch.empty(max(nb, 4), dtype=torch.uint8, device="cuda")
    swl.kv4_evict_device(c.desc(), b, keep, d_weights=w.data_ptr(), weights_stride=w.stride(1), d_dst_table=dst.data_ptr(),
                         dst_stride=per, d_new_lens=nl.data_ptr(), first=first, recent=recent,
                         d_new_weights=nw.data_ptr() if with_weights else 0, new_weights_stride=most + 3 if with_weights else 0,
                         d_kept=kept.data_ptr() if with_kept else 0, kept_stride=most + 2 if with_kept else 0,
                         d_work=0 if with_kept else work.data_ptr(), work_bytes=0 if with_kept else nb)
    torch.cuda.synchronize()
    return dst, nl, kept, nw


def check_evict(c, lens, w, keep, first, recent, **kw):
    torch, _ = _torch()
    dst, nl, kept, nw = run_evict(c, lens, w, keep, first, recent, **kw)
    wn = w.cpu().numpy()
    held = np.full((2, c.nseq, max(1, min(keep, c.max_len)), c.kvh, c.hd), np.nan, np.float32)
    for i, n in enumerate(lens):
        m = min(n, keep)
        assert int(nl[i]) == m
        for h in range(c.kvh):
            s = survivors(wn[i, h], n, keep, first, recent)
            if kw.get("with_kept", True):
                assert np.array_equal(kept[i, h, :m].cpu().numpy(), s), (i, h)
                assert (kept[i, h, m:] == -9).all()
            if kw.get("with_weights", True):
                assert np.array_equal(nw[i, h, :m].cpu().numpy(), wn[i, h, s], equal_nan=True) and (nw[i, h, m:] == -9).all()
            held[:, i, :m, h] = c.held[:, i, s, h]
        if m:
            x = torch.zeros(2, m, c.kvh, c.hd, device="cuda")
            one = swl.swl_kv4_cache(c.pool.data_ptr(), dst[i:].data_ptr(), dst.stride(0), c.num, c.page, c.kvh, c.hd, c.group)
            b = c.batch([m], [m])
            b.max_len = m
            swl.kv4_read_device(one, b, x[0].data_ptr(), x[1].data_ptr())
            torch.cuda.synchronize()
            assert np.array_equal(x.cpu().numpy(), held[:, i, :m])
    assert int(c.status) == 0
    return dst, nl, nw, held


@pytest.mark.parametrize("keep,first,recent", [(64, 4, 16), (64, 0, 0), (64, 32, 32), (63, 63, 0), (1, 0, 0), (129, 5, 100), (0, 0, 0), (500, 4, 4)])
@pytest.mark.parametrize("kvh,hd,group,page", [(2, 256, 64, 64), (3, 64, 64, 16), (1, 128, 128, 128)])
def test_evict(kvh, hd, group, page, keep, first, recent):
    torch, _ = _torch()
    rng = np.random.default_rng(keep + hd)
    lens = [300, 64, 65, 0, 1, 129, 130]
    c = Cache(7, 300, kvh, hd, group, page, spare=7 * (-(-300 // page)))
    c.fill(lens, rng)
    w = torch.from_numpy(rng.random((7, kvh, 305)).astype(np.float32) ** 4).cuda()
    check_evict(c, lens, w, keep, first, recent)


@pytest.mark.parametrize("kind", ["all equal", "few values", "zeros", "nan", "negative", "infinite"])
def test_evict_ties_and_odd_weights(kind):
    torch, _ = _torch()
    rng = np.random.default_rng(1)
    c = Cache(2, 2600, 2, 64, page=32, spare=200)
    lens = [2600, 1500]
    c.fill(lens, rng)
    w = rng.random((2, 2, 2600)).astype(np.float32)
    if kind == "all equal":
        w[:] = 0.5
    elif kind == "few values":
        w = np.floor(w * 3).astype(np.float32)
    elif kind == "zeros":
        w = np.where(w < 0.5, np.float32(0.0), np.float32(-0.0))
    elif kind == "nan":
        w[w < 0.6] = np.nan
        w[w > 0.9] = -np.inf
    elif kind == "negative":
        w = w - np.float32(0.5)
    else:
        w[w > 0.3] = np.inf
    check_evict(c, lens, torch.from_numpy(w).cuda(), 1111, 3, 200)


def test_evict_long():
    """Lengths that are spread over several blocks."""
    torch, _ = _torch()
    rng = np.random.default_rng(2)
    c = Cache(2, 40000, 1, 64, page=128, spare=400)
    lens = [40000, 20001]
    c.fill(lens, rng)
    w = torch.from_numpy((rng.random((2, 1, 40000)) ** 6).astype(np.float32)).cuda()
    check_evict(c, lens, w, 19999, 4, 512)


def test_evict_without_optional_outputs():
    torch, _ = _torch()
    rng = np.random.default_rng(3)
    c = Cache(2, 200, 2, 128, spare=8)
    c.fill([200, 150], rng)
    w = torch.from_numpy(rng.random((2, 2, 200)).astype(np.float32)).cuda()
    check_evict(c, [200, 150], w, 100, 2, 10, with_kept=False, with_weights=False)


def test_conversation():
    """The calls as a server makes them: prompt, steps that accumulate weights, eviction into fresh pages, further steps."""
    torch, _ = _torch()
    rng = np.random.default_rng(9)
    c = Cache(3, 260, 2, 256, spare=3 * 4)
    lens = [150, 90, 200]
    c.append(lens, lens, rng)
    w = torch.zeros(3, 2, 260, device="cuda")
    got, lse, q = attend(c, lens, lens, 8, rng, gate=True, weights=w)
    check(c, lens, lens, 8, got, lse, q, gate=True, weights=w.cpu().numpy().astype(np.float64), before=np.zeros((3, 2, 260)))
    for _ in range(4):
        lens = [m + 1 for m in lens]
        c.append(lens, [1, 1, 1], rng)
        before = w.cpu().numpy().astype(np.float64)
        got, lse, q = attend(c, lens, [1, 1, 1], 8, rng, gate=True, weights=w)
        check(c, lens, [1, 1, 1], 8, got, lse, q, gate=True, weights=w.cpu().numpy().astype(np.float64), before=before)
    dst, nl, nw, held = check_evict(c, lens, w, 128, 4, 32)
    lens = [int(x) for x in nl]
    assert lens == [128, 94, 128]
    # on with the evicted cache (its tables end two pages further)
    c2 = Cache(3, 256, 2, 256)
    c2.pool, c2.num = c.pool, c.num
    c2.table = torch.cat([dst, torch.from_numpy(c.spare[6:12].reshape(3, 2).copy()).cuda()], 1).contiguous()
    c2.held[:, :, :128] = held
    w2 = torch.zeros(3, 2, 256, device="cuda")
    w2[..., :128] = nw[..., :128]
    for new in ([1, 1, 1], [30, 1, 7]):
        lens = [m + n for m, n in zip(lens, new)]
        c2.append(lens, new, rng)
        before = w2.cpu().numpy().astype(np.float64)
        got, lse, q = attend(c2, lens, new, 8, rng, weights=w2)
        check(c2, lens, new, 8, got, lse, q, weights=w2.cpu().numpy().astype(np.float64), before=before)
