"""The 4-bit KV cache operators as they are measured: writing tokens into the
cache (and reading them back), attention over it for single tokens and for
prompts, with and without the accumulation of attention weights, and eviction
by those weights. With ``own`` false ``run`` computes them with elementary
torch operations; with ``own`` true it calls swiftlet_b200."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODE = {"f32": 0, "bf16": 1, "f16": 2}
# kv_heads 2, rep 8, head_dim 256 is the attention of the 35B and 80B
# configurations, kv_heads 2, rep 2, head_dim 128 that of the MID one; the
# others are generic grouped, multi-query and multi-head layouts.
HEADS = [(2, 8, 256), (2, 8, 256), (2, 2, 128), (4, 4, 128), (8, 4, 128), (1, 8, 64), (8, 1, 64), (2, 6, 128), (1, 16, 128)]


def _case(name, op, dtype, nseq, len_lo, len_hi, new_lo, new_hi, kv_heads=2, rep=8, hd=256, group=64, page=64, weights=False,
          gate=False, keep=0, first=0, recent=0):
    c = dict(op=op, dtype=dtype, nseq=nseq, len_lo=len_lo, len_hi=len_hi, new_lo=new_lo, new_hi=new_hi, kv_heads=kv_heads, rep=rep,
             hd=hd, group=group, page=page, weights=weights, gate=gate, keep=keep, first=first, recent=recent)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # a decode step of a full batch: one new token per conversation
        _case("append_step", "append", "f32", 64, 100, 8000, 1, 1),
        # prompts of several new conversations written at once, ragged
        _case("append_prompts", "append", "bf16", 9, 2500, 9001, 2500, 9001),
        # one conversation, short: the latency of a single token
        _case("attend_one_short", "attention", "f32", 1, 777, 777, 1, 1, gate=True),
        # one conversation, very long: the context is split over the GPU
        _case("attend_one_long", "attention", "f32", 1, 131072, 131072, 1, 1, gate=True),
        # a full batch of conversations of mixed length, with the gate of the model's attention
        _case("attend_batch", "attention", "f32", 64, 61, 8192, 1, 1, gate=True),
        # a full batch of long conversations
        _case("attend_batch_long", "attention", "bf16", 64, 20000, 32768, 1, 1),
        # a batch that accumulates the weights by which it later evicts
        _case("attend_weights", "attention", "f32", 16, 3000, 8200, 1, 1, weights=True),
        # a launch of prompt chunks on running conversations, ragged
        _case("attend_chunks", "attention", "f32", 8, 900, 4100, 33, 200, gate=True),
        # a long new turn on a longer conversation
        _case("attend_turn", "attention", "bf16", 1, 10000, 10000, 2048, 2048, gate=True),
        # a prompt from its first token, smaller heads, small pages
        _case("attend_prompt", "attention", "f16", 1, 8192, 8192, 8192, 8192, kv_heads=4, rep=4, hd=128, group=128, page=16),
        # one very long conversation cut to half
        _case("evict_one_long", "evict", "f32", 1, 65536, 65536, 0, 0, keep=32768, first=4, recent=256),
        # a batch trimmed back to its budget
        _case("evict_batch", "evict", "f32", 64, 1500, 4608, 0, 0, keep=4096, first=4, recent=512),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "step", "step", "prompt", "prompt", "evict"])
    kvh, rep, hd = rng.choice(HEADS)
    group = rng.choice([g for g in (64, 128) if g <= hd])
    page = rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["f32", "bf16", "f16"])
    h = dict(kv_heads=kvh, rep=rep, hd=hd, group=group, page=page)
    most = 2 ** 28 // (kvh * hd)  # slots in all: about a quarter of the largest listed case
    if op == "append":
        n = _log(rng, 1, 8192)
        nseq = _log(rng, 1, max(1, min(64, 40000 // n)))
        lo = max(1, int(n * rng.uniform(0.2, 1)))
        extra = _log(rng, 1, 4000)
        return _case("", "append", dtype, nseq, n + extra // 3, n + extra, lo, n, **h)
    if op == "step":
        nseq = _log(rng, 1, 96)
        hi = _log(rng, 1, max(2, min(100000, most // nseq)))
        return _case("", "attention", dtype, nseq, max(1, int(hi * rng.uniform(0.02, 1))), hi, 1, 1, weights=rng.random() < 0.3,
                     gate=rng.random() < 0.5, **h)
    if op == "prompt":
        nseq = _log(rng, 1, 12)
        n = _log(rng, 2, 1500 // nseq)
        hi = n + _log(rng, 1, 6000)
        return _case("", "attention", dtype, nseq, n, hi, max(1, n // 3), n, weights=rng.random() < 0.3, gate=rng.random() < 0.5, **h)
    nseq = _log(rng, 1, 64)
    hi = _log(rng, 40, max(80, min(60000, most // 4 // nseq)))
    keep = max(20, int(hi * rng.uniform(0.3, 0.95)))
    return _case("", "evict", "f32", nseq, max(1, hi // 3), hi, 0, 0, keep=keep, first=rng.choice([0, 4]), recent=rng.randint(0, keep // 4), **h)


def _spread(lo, hi, n, odd):
    """n whole numbers from hi down to lo in a scattered order (a function of the case alone)."""
    return [hi if n == 1 else hi - (hi - lo) * ((i * odd) % n) // (n - 1) for i in range(n)]


def _lengths(case):
    n = case["nseq"]
    new = _spread(case["new_lo"], case["new_hi"], n, 5 if n % 5 else 3 if n % 3 else 1)
    lens = [max(a, b) for a, b in zip(_spread(case["len_lo"], case["len_hi"], n, 7 if n % 7 else 3 if n % 3 else 1), new)]
    return lens, new


def _row_bytes(case):
    return case["hd"] // 2 + 4 * (case["hd"] // case["group"])


def _page_bytes(case):
    return case["kv_heads"] * 2 * case["page"] * _row_bytes(case)


def work(case):
    lens, new = _lengths(case)
    kvh, hd, rep = case["kv_heads"], case["hd"], case["rep"]
    e = 4 if case["dtype"] == "f32" else 2
    row = 2 * kvh * _row_bytes(case)  # one slot's keys and values
    if case["op"] == "append":  # rows in, cache written, cache read, rows out
        return {"bytes": sum(new) * (2 * 2 * kvh * hd * e + 2 * row), "flops": 0}
    if case["op"] == "evict":
        kept = sum(min(n, case["keep"]) for n in lens)
        return {"bytes": sum(lens) * kvh * 4 + kept * (2 * row + kvh * 8), "flops": 0}
    seen = sum(n * (m - n) + n * (n + 1) // 2 for m, n in zip(lens, new))
    b = sum(lens) * row + sum(new) * kvh * rep * hd * e * (3 if case["gate"] else 2) + sum(new) * kvh * rep * 4
    if case["weights"]:
        b += sum(lens) * kvh * 8
    return {"bytes": b, "flops": 4 * seen * kvh * rep * hd}


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    lens, new = _lengths(case)
    nseq, kvh, hd, page, group = case["nseq"], case["kv_heads"], case["hd"], case["page"], case["group"]
    H, dt = kvh * case["rep"], DTYPES[case["dtype"]]
    i32 = dict(dtype=torch.int32, device=dev)

    def rows(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device=dev) * scale).to(dtype)

    per = [-(-n // page) for n in lens]
    stride = max(per)
    dst_per = [-(-min(n, case["keep"]) // page) for n in lens] if case["op"] == "evict" else [0] * nseq
    dst_stride = max(max(dst_per), 1)
    num_pages = sum(per) + sum(dst_per) + 1
    order = torch.randperm(num_pages, generator=g, device=dev).to(torch.int32)

    def table(counts, width, base):
        t = torch.zeros(nseq, width, **i32)
        for i, c in enumerate(counts):
            t[i, :c] = order[base:base + c]
            base += c
        return t

    s = {"case": dict(case), "nseq": nseq, "kvh": kvh, "hd": hd, "page": page, "group": group, "H": H, "num_pages": num_pages,
         "max_len": max(lens), "max_new": max(new), "total": sum(new), "keep": case["keep"], "max_keep": max(min(n, case["keep"]) for n in lens),
         "table": table(per, stride, 0), "lens": torch.tensor(lens, **i32),
         "start": torch.tensor([sum(new[:i]) for i in range(nseq + 1)], **i32)}
    # pages as they stand after many writes: codes over the whole range, keys and values of unit size about
    seg = min(page, 64)
    blk = seg * _row_bytes(case)
    pool = torch.randint(0, 256, (num_pages * kvh * (page // seg) * 2, blk), generator=g, device=dev, dtype=torch.uint8)
    params = pool[:, seg * hd // 2:].view(torch.float16).view(pool.shape[0], -1, 2)
    spread = torch.rand(params.shape[:2], generator=g, device=dev)
    params[..., 0] = (0.2 + 0.2 * spread).half()
    params[..., 1] = (-7.5 * (0.2 + 0.2 * spread) + 0.3 * (torch.rand(spread.shape, generator=g, device=dev) - 0.5)).half()
    s["pool"] = pool.view(-1)
    wstride = max(lens) + 5
    if case["op"] == "append":
        # keys with a few large channels, as after rotation; values without
        big = 1.0 + 4.0 * (torch.rand(kvh, hd, generator=g, device=dev) > 0.97)
        s["k"], s["v"] = (torch.randn(s["total"], kvh, hd, generator=g, device=dev) * big).to(dt), rows(s["total"], kvh, hd)
        s["k_back"], s["v_back"] = torch.empty_like(s["k"]), torch.empty_like(s["v"])
    elif case["op"] == "attention":
        s["scale"] = 1.0 / math.sqrt(hd)
        s["q"] = rows(s["total"], H, hd, scale=1.2)
        s["gate"] = rows(s["total"], H, hd) if case["gate"] else None
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(s["total"], H, device=dev)
        s["weights"] = torch.rand(nseq, kvh, wstride, generator=g, device=dev) if case["weights"] else None
    else:
        # weights as they accumulate: a few slots hold much, most hold little
        s["weights"] = torch.rand(nseq, kvh, wstride, generator=g, device=dev).clamp_min(1e-6).pow(6) * 20
        s["dst_table"] = table(dst_per, dst_stride, sum(per))
        s["first"], s["recent"] = case["first"], case["recent"]
        s["new_lens"] = torch.zeros(nseq, **i32)
        s["kept"] = torch.full((nseq, kvh, s["max_keep"]), -1, **i32)
        s["new_weights"] = torch.zeros(nseq, kvh, s["max_keep"], device=dev)
    return s


# ------------------------------------------------------------ plain forms --
def _swizzle(hd, slots):
    """XOR on the position of a row's units (8 of them) by the slot in its block."""
    if hd == 256:
        return (slots & 6) ^ ((slots & 1) << 2)
    return (slots & 2) << 1 if hd == 128 else torch.zeros_like(slots)


def _unit_order(s):
    t = torch.arange(min(s["page"], 64), device="cuda")
    return torch.arange(8, device="cuda")[None, :] ^ _swizzle(s["hd"], t)[:, None]


def _blocks(s):
    """The pool as [page][head][block][K, V][bytes of a block's keys or values]."""
    seg = min(s["page"], 64)
    return s["pool"].view(s["num_pages"], s["kvh"], s["page"] // seg, 2, seg * (s["hd"] // 2 + 4 * (s["hd"] // s["group"])))


def _values(s, table):
    """Keys and values of every slot of every sequence of a table: [2][nseq][kvh][slots][hd] in 32 bits."""
    hd, ng, seg = s["hd"], s["hd"] // s["group"], min(s["page"], 64)
    b = _blocks(s)[table.long()].permute(4, 0, 2, 1, 3, 5)  # [2][nseq][kvh][pages][blocks][bytes]
    lead = b.shape[:5]
    codes = b[..., :seg * hd // 2].reshape(*lead, seg, 8, hd // 16)
    codes = torch.gather(codes, 6, _unit_order(s)[:, :, None].expand(*lead, seg, 8, hd // 16))
    nib = torch.stack((codes & 15, codes >> 4), -1).view(*lead, seg, 8, hd // 64, 8)  # unit r, word w, code: channel 64 w + 8 r + code
    q = nib.transpose(-3, -2).reshape(*lead, seg, ng, hd // ng).float()
    p = b[..., seg * hd // 2:].contiguous().view(torch.float16).view(*lead, seg, ng, 2).float()
    return (q * p[..., 0:1] + p[..., 1:2]).view(2, lead[1], lead[2], -1, hd)


def _tokens(s):
    """Per row of the token buffers: its sequence and its slot."""
    j = torch.arange(s["total"], device="cuda")
    seq = torch.searchsorted(s["start"].long(), j, right=True) - 1
    n = (s["start"][1:] - s["start"][:-1]).long()
    return seq, s["lens"].long()[seq] - n[seq] + j - s["start"].long()[seq]


def _plain_append(s):
    hd, ng, seg = s["hd"], s["hd"] // s["group"], min(s["page"], 64)
    seq, slot = _tokens(s)
    x = torch.stack((s["k"], s["v"])).float().view(2, s["total"], s["kvh"], ng, -1)
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    b, sc = lo.half(), ((hi - lo) * (1.0 / 15.0)).half()
    inv = torch.where(sc.float() > 0, 1.0 / sc.float(), torch.zeros_like(lo))
    q = ((x - b.float()) * inv).round().clamp(0, 15).to(torch.uint8).view(2, s["total"], s["kvh"], hd // 64, 8, 4, 2)
    units = (q[..., 0] | (q[..., 1] << 4)).transpose(3, 4)  # unit r, word w, byte
    order = _unit_order(s)[slot % seg]
    units = torch.gather(units, 3, order[None, :, None, :, None, None].expand_as(units)).reshape(2, s["total"], s["kvh"], hd // 2)
    params = torch.cat((sc, b), -1).view(torch.uint8).reshape(2, s["total"], s["kvh"], 4 * ng)
    pg, blk, t = s["table"].long()[seq, slot // s["page"]], slot % s["page"] // seg, slot % seg
    pool = _blocks(s)
    codes = pool[..., :seg * hd // 2].view(*pool.shape[:4], seg, hd // 2)
    pars = pool[..., seg * hd // 2:].view(*pool.shape[:4], seg, 4 * ng)
    heads, kv = torch.arange(s["kvh"], device="cuda"), torch.arange(2, device="cuda")
    at = (pg[None, :, None], heads[None, None, :], blk[None, :, None], kv[:, None, None], t[None, :, None])
    codes[at] = units
    pars[at] = params
    back = (q.reshape(2, s["total"], s["kvh"], ng, -1).float() * sc.float() + b.float()).view(2, s["total"], s["kvh"], hd).to(s["k"].dtype)
    return {"k": back[0], "v": back[1]}


def _plain_attention(s):
    kvh, hd, rep, n = s["kvh"], s["hd"], s["H"] // s["kvh"], s["max_new"]
    kv = _values(s, s["table"])
    L = kv.shape[3]
    seq, slot = _tokens(s)
    at = seq * n + torch.arange(s["total"], device="cuda") - s["start"].long()[seq]
    q = torch.zeros(s["nseq"] * n, kvh, rep, hd, device="cuda")
    q[at] = s["q"].float().view(-1, kvh, rep, hd)
    q = q.view(s["nseq"], n, kvh, rep, hd).permute(0, 2, 1, 3, 4).reshape(s["nseq"], kvh, n * rep, hd)
    last = torch.full((s["nseq"] * n,), -1, dtype=torch.long, device="cuda")
    last[at] = slot
    seen = torch.arange(L, device="cuda") <= last.view(s["nseq"], 1, n, 1)
    # what no row sees is unwritten memory: it must not reach the products
    there = torch.arange(L, device="cuda") < s["lens"].long()[:, None]
    kv = torch.where(there[None, :, None, :, None], kv, torch.zeros((), device="cuda"))
    x = (q @ kv[0].transpose(-1, -2) * s["scale"]).view(s["nseq"], kvh, n, rep, L)
    x = x.masked_fill(~seen[:, :, :, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    e = (x - top.clamp_min(-1e30)).exp()
    total = e.sum(-1, keepdim=True)
    p = e / total.clamp_min(1e-30)
    o = (p.view(s["nseq"], kvh, n * rep, L) @ kv[1]).view(s["nseq"], kvh, n, rep, hd).permute(0, 2, 1, 3, 4).reshape(-1, s["H"], hd)[at]
    lse = (top + total.log()).permute(0, 2, 1, 3, 4).reshape(-1, s["H"])[at]
    if s["gate"] is not None:
        o = o / (1.0 + (-s["gate"].float()).exp())
    r = {"out": o.to(s["q"].dtype), "lse": lse}
    if s["weights"] is not None:
        s["weights"][..., :L] += p.sum((2, 3))[..., :s["weights"].shape[-1]]
        r["weights"] = s["weights"]
    return r


def _plain_evict(s):
    lens, L = s["lens"].long()[:, None], s["max_len"]
    slot = torch.arange(L, device="cuda")[None, None, :]
    there = slot < lens[:, None]
    w = s["weights"][..., :L]
    w = torch.where(torch.isnan(w), torch.full_like(w, -math.inf), w)
    new_lens = s["lens"].clamp_max(s["keep"])
    # order: the protected first, then by weight, then by slot
    rank = w.argsort(dim=-1, descending=True, stable=True)
    held = ((slot < s["first"]) | (slot >= lens[:, None] - s["recent"])).long() + 2 * there.long()
    rank = rank.gather(-1, held.expand_as(w).gather(-1, rank).argsort(dim=-1, descending=True, stable=True))
    place = torch.empty_like(rank).scatter_(-1, rank, slot.expand_as(rank))
    chosen = there & (place < new_lens.long()[:, None, None])
    i, h, t = chosen.nonzero(as_tuple=True)
    to = (chosen.cumsum(-1) - 1)[i, h, t]
    s["kept"][i, h, to] = t.to(torch.int32)
    s["new_weights"][i, h, to] = s["weights"][i, h, t]
    s["new_lens"].copy_(new_lens)
    seg, hd = min(s["page"], 64), s["hd"]
    pool = _blocks(s)
    codes = pool[..., :seg * hd // 2].view(*pool.shape[:4], seg, 8, hd // 16)
    pars = pool[..., seg * hd // 2:].view(*pool.shape[:4], seg, -1)
    src = (s["table"].long()[i, t // s["page"]], h, t % s["page"] // seg)
    dst = (s["dst_table"].long()[i, to // s["page"]], h, to % s["page"] // seg)
    order = _unit_order(s)
    # a row's units stand in another order in another slot: undo the source's, apply the destination's
    units = codes[src[0], src[1], src[2], :, t % seg]
    mix = order[t % seg].gather(1, order[to % seg])
    codes[dst[0], dst[1], dst[2], :, to % seg] = units.gather(2, mix[:, None, :, None].expand_as(units))
    pars[dst[0], dst[1], dst[2], :, to % seg] = pars[src[0], src[1], src[2], :, t % seg]
    return {"kept": s["kept"], "weights": s["new_weights"], "lens": s["new_lens"], "pages": s["pool"]}


# -------------------------------------------------------- the framework's --
def _handles(s):
    """What a program keeps beside its buffers: the cache and batch descriptors and the workspace."""
    import swiftlet_b200 as swl
    p = lambda k: s[k].data_ptr() if s.get(k) is not None else 0  # noqa: E731
    s["cache"] = swl.swl_kv4_cache(p("pool"), p("table"), s["table"].stride(0), s["num_pages"], s["page"], s["kvh"], s["hd"], s["group"])
    s["batch"] = swl.swl_kv4_batch(p("start"), p("lens"), s["nseq"], s["total"], s["max_new"], s["max_len"])
    if s["case"]["op"] == "attention":
        n = swl.kv4_attention_workspace(s["cache"], s["batch"], s["H"])
        s["work"] = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
    elif s["case"]["op"] == "evict":
        n = swl.kv4_evict_workspace(s["cache"], s["batch"], s["keep"])
        s["work"] = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")


def _own(s):
    import swiftlet_b200 as swl
    if "cache" not in s:
        _handles(s)
    p = lambda k: s[k].data_ptr() if s.get(k) is not None else 0  # noqa: E731
    stream, dt = torch.cuda.current_stream().cuda_stream, CODE[s["case"]["dtype"]]
    if s["case"]["op"] == "append":
        swl.kv4_append_device(s["cache"], s["batch"], p("k"), p("v"), dtype=dt, stream=stream)
        swl.kv4_read_device(s["cache"], s["batch"], p("k_back"), p("v_back"), dtype=dt, stream=stream)
        return {"k": s["k_back"], "v": s["v_back"]}
    if s["case"]["op"] == "attention":
        w = s["weights"]
        swl.kv4_attention_device(s["cache"], s["batch"], s["H"], p("q"), p("out"), dtype=dt, scale=s["scale"], d_gate=p("gate"),
                                 d_lse=p("lse"), d_weights=p("weights"), weights_stride=0 if w is None else w.stride(1),
                                 d_work=p("work"), work_bytes=s["work"].numel(), stream=stream)
        r = {"out": s["out"], "lse": s["lse"]}
        if w is not None:
            r["weights"] = w
        return r
    swl.kv4_evict_device(s["cache"], s["batch"], s["keep"], d_weights=p("weights"), weights_stride=s["weights"].stride(1),
                         d_dst_table=p("dst_table"), dst_stride=s["dst_table"].stride(0), first=s["first"], recent=s["recent"],
                         d_new_lens=p("new_lens"), d_new_weights=p("new_weights"), new_weights_stride=s["new_weights"].stride(1),
                         d_kept=p("kept"), kept_stride=s["kept"].stride(1), d_work=p("work"), work_bytes=s["work"].numel(), stream=stream)
    return {"kept": s["kept"], "weights": s["new_weights"], "lens": s["new_lens"], "pages": s["pool"]}


def run(state):
    if own:
        return _own(state)
    return {"append": _plain_append, "attention": _plain_attention, "evict": _plain_evict}[state["case"]["op"]](state)


# ----------------------------------------------------------------- exact --
def _look_up(s, i, h, which, slots):
    """Values of sequence i, kv head h at some slots by the address of each channel's code, in 64 bits."""
    hd, group, page = s["hd"], s["group"], s["page"]
    seg, ng = min(page, 64), hd // group
    row = hd // 2 + 4 * ng
    ch = torch.arange(hd, device="cuda")
    t = slots % seg
    base = ((s["table"][i].long()[slots // page] * s["kvh"] + h) * (page // seg) + slots % page // seg) * 2 * seg * row + which * seg * row
    unit = (ch % 64 // 8)[None, :] ^ _swizzle(hd, t)[:, None]
    byte = base[:, None] + t[:, None] * (hd // 2) + unit * (hd // 16) + (ch // 64 * 4 + ch % 8 // 2)[None, :]
    code = (s["pool"][byte] >> (4 * (ch % 2)).to(torch.uint8)) & 15
    half = s["pool"].view(torch.float16)
    par = (base[:, None] + seg * (hd // 2) + 4 * (t[:, None] * ng + (ch // group)[None, :])) // 2
    return half[par].double() * code.double() + half[par + 1].double()


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "evict":
        return None  # rows and weights are moved, not computed
    if case["op"] == "append":
        # the definition of a code names its roundings to 32 bits: each is made here, and nothing else is rounded
        out = []
        for x in (s["k"], s["v"]):
            y = x.double().view(s["total"], s["kvh"], -1, s["group"])
            lo, hi = y.min(-1, keepdim=True).values, y.max(-1, keepdim=True).values
            fifteenth = torch.tensor(1 / 15, device="cuda").double()
            b, sc = lo.half().double(), ((hi - lo).float().double() * fifteenth).float().half().double()
            inv = (1 / sc).float().double()
            code = torch.round(((y - b).float().double() * inv).float().double()).clamp(0, 15)
            out.append((code * sc + b).view(x.shape))
        return {"k": out[0], "v": out[1]}
    lens, new = _lengths(case)
    rep = case["rep"]
    o = torch.empty(s["total"], s["H"], s["hd"], dtype=torch.float64, device="cuda")
    lse = torch.empty(s["total"], s["H"], dtype=torch.float64, device="cuda")
    w = None if s["weights"] is None else s["weights"].double()
    a = 0
    for i, (m, n) in enumerate(zip(lens, new)):
        slots = torch.arange(m, device="cuda")
        hidden = slots[None, :] > torch.arange(m - n, m, device="cuda")[:, None]
        for h in range(s["kvh"]):
            k, v = _look_up(s, i, h, 0, slots), _look_up(s, i, h, 1, slots)
            for r in range(rep):
                x = s["q"][a:a + n, h * rep + r].double() @ k.T * s["scale"]
                x[hidden] = -math.inf
                z = torch.logsumexp(x, -1)
                p = torch.exp(x - z[:, None])
                o[a:a + n, h * rep + r], lse[a:a + n, h * rep + r] = p @ v, z
                if w is not None:
                    w[i, h, :m] += p.sum(0)
        a += n
    if s["gate"] is not None:
        o *= torch.sigmoid(s["gate"].double())
    r = {"out": o, "lse": lse}
    if w is not None:
        r["weights"] = w
    return r
