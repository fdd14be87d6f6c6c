"""The operators of a prompt with several position axes: multi-axis positions, the rotary K/V write, whole-prompt
attention.  A case is one call of one operator; `run` makes it, in elementary torch operations or (`own`) through the
framework.

  positions  iian_pa_mrope_positions: positions on three axes and attendable cells of a step's new tokens, from each
             request's runs of text and grids of image or video patches
  rope       iian_pa_mrope_kv_write: q and K rotated (after the heads' RMS norm where the model has one), K and V
             written into the paged pool
  attn       iian_pa_prompt_attention: attention over packed prompts of different lengths

Lengths and grids are drawn from `lens_seed`, so they belong to the case; values come from the seed.  Calls are bound to
their buffers once, as an engine that holds its arguments makes them.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
POOL_TYPES = {"f32": 0, "f16": 1, "q8_0": 8}
ELEM = {"f32": 4.0, "f16": 2.0, "bf16": 2.0, "q8_0": 34.0 / 32.0}
BS = 16           # cells per block of the pool
EPS = 1e-6


def _attn(name, type_, H, Hkv, D, S, lo, hi, **kw):
    c = dict(name=name, op="attn", type=type_, H=H, Hkv=Hkv, D=D, S=S, lo=lo, hi=hi, causal=True, n_swa=0, softcap=0.0,
             images=False, fused=False, lens_seed=1)
    c.update(kw)
    return c


def _rope(name, type_, H, Hkv, D, T, **kw):
    c = dict(name=name, op="rope", type=type_, H=H, Hkv=Hkv, D=D, T=T, pool="f16", norm=False, layout="sections",
             neox=True, fused=False, pos_hi=32768, lens_seed=1)
    c.update(kw)
    return c


def _positions(name, S, T, spans, **kw):
    c = dict(name=name, op="positions", S=S, T=T, spans=spans, full=False, lens_seed=1)
    c.update(kw)
    return c


def listed():
    return [
        # a few short questions at once, a small model: launches and latency
        _attn("attn_short", "bf16", 14, 2, 64, 4, 1, 64, lens_seed=1),
        # new prompts of an 8B model, ragged, read out of the fused projection's rows
        _attn("attn_ragged", "bf16", 32, 8, 128, 16, 100, 2000, fused=True, lens_seed=2),
        # one long prompt of that model
        _attn("attn_long", "f16", 32, 8, 128, 1, 8192, 8192, lens_seed=3),
        # two prompts in full precision, as an engine whose rows are f32 has them
        _attn("attn_f32", "f32", 32, 8, 128, 2, 300, 1100, lens_seed=4),
        # a vision tower: images of some hundred to two thousand patches, every patch sees its image
        _attn("attn_vision", "bf16", 16, 16, 80, 6, 400, 2100, causal=False, lens_seed=5),
        # a sliding-window layer at head size 256, prompts with images whose patches see their whole image
        _attn("attn_window", "bf16", 16, 8, 256, 3, 1500, 4000, n_swa=1024, images=True, softcap=50.0, lens_seed=6),
        # a decode step: one token per sequence, f32 rows
        _rope("rope_decode", "f32", 32, 8, 128, 64, lens_seed=7),
        # a prompt step of a model with normed heads, interleaved axes, out of the fused projection's rows
        _rope("rope_prompt", "bf16", 32, 8, 128, 1903, norm=True, layout="interleaved", fused=True, lens_seed=8),
        # a quantised pool
        _rope("rope_q8", "f32", 32, 8, 128, 889, pool="q8_0", neox=False, lens_seed=9),
        # a long video prompt in one step, far positions
        _rope("rope_long", "f16", 16, 8, 256, 16384, norm=True, pos_hi=1000000, lens_seed=10),
        # running decodes of multimodal requests
        _positions("positions_decode", 48, 48, 12, lens_seed=11),
        # prompts with hours of video: some thousand frames, each behind its time stamp
        _positions("positions_video", 4, 131072, 2000, full=True, lens_seed=12),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(32, 8, 128), (14, 2, 64), (9, 3, 64), (28, 4, 128), (16, 16, 80), (20, 20, 96), (16, 8, 256), (40, 8, 128),
         (8, 1, 72), (12, 12, 64)]


def draw(rng):
    """One more case of the ranges that the listed ones stand for."""
    seed = rng.randrange(1 << 30)
    op = rng.choice(["attn", "attn", "rope", "positions"])
    if op == "attn":
        H, Hkv, D = rng.choice(HEADS)
        t = rng.choice(["bf16", "bf16", "f16", "f32"])
        hi = _log_int(rng, 1, 8192 if t != "f32" else 2048)
        # what the padded plain form computes stays below one prompt of 8192 tokens at 32 heads of 128
        most = 32 * 128 * 8192 ** 2 // (6 if t == "f32" else 1)
        S = max(1, min(_log_int(rng, 1, 48), most // (H * D * hi * hi)))
        causal = rng.random() < 0.7
        return dict(op="attn", type=t, H=H, Hkv=Hkv, D=D, S=S, lo=rng.choice([hi, max(1, hi // 8), 1]), hi=hi,
                    causal=causal, n_swa=rng.choice([0, 0, 0, 128, 1000]), softcap=rng.choice([0.0, 0.0, 0.0, 30.0]),
                    images=causal and rng.random() < 0.3, fused=rng.random() < 0.5, lens_seed=seed)
    if op == "rope":
        H, Hkv, D = rng.choice(HEADS)
        pool = rng.choice(["f16", "f16", "f32", "q8_0"] if D % 32 == 0 else ["f16", "f32"])
        T = _log_int(rng, 1, 16384 * 32 * 128 // ((H + 2 * Hkv) * D))
        return dict(op="rope", type=rng.choice(["f32", "f16", "bf16"]), H=H, Hkv=Hkv, D=D, T=T, pool=pool,
                    norm=rng.random() < 0.5, layout=rng.choice(["sections", "interleaved", "restart"]),
                    neox=rng.random() < 0.7, fused=rng.random() < 0.5, pos_hi=rng.choice([4096, 131072, 1000000]),
                    lens_seed=seed)
    S = _log_int(rng, 1, 64)
    return dict(op="positions", S=S, T=_log_int(rng, S, 131072), spans=_log_int(rng, 1, 2000), full=rng.random() < 0.5,
                lens_seed=seed)


# ---- the lengths of a case ----

def _lens(c):
    r = np.random.RandomState(c["lens_seed"] % (1 << 31))
    n = np.exp(r.uniform(math.log(c["lo"]), math.log(c["hi"] + 0.999), c["S"])).astype(np.int64).clip(c["lo"], c["hi"])
    n[r.randint(c["S"])] = c["hi"]
    return n


def _row_end(c, lens):
    """Of each token, the cells of its own prompt that it may attend: those up to itself, and all of its image."""
    r = np.random.RandomState((c["lens_seed"] + 1) % (1 << 31))
    ends = []
    for n in lens:
        e = np.arange(1, n + 1)
        a = int(r.randint(0, 40))
        while a < n:
            b = min(n, a + int(r.randint(16, 300)))
            e[a:b] = b
            a = b + int(r.randint(1, 400))
        ends.append(e)
    return np.concatenate(ends).astype(np.int32)


def _visible(c, lens, ends):
    """(head-independent) pairs of a token and a cell that it attends."""
    total, o = 0, 0
    for n in lens:
        i = np.arange(n)
        hi = ends[o:o + n].astype(np.int64) if ends is not None else i + 1 if c["causal"] else np.full(n, n)
        lo = np.maximum(0, i - c["n_swa"] + 1) if c["n_swa"] else np.zeros(n, np.int64)
        total += int(np.maximum(0, hi - lo).sum())
        o += n
    return total


def _spans(c):
    """int32 [N, 4] spans of all requests, their offsets, and the computed and new tokens of each request."""
    r = np.random.RandomState(c["lens_seed"] % (1 << 31))
    S, T = c["S"], c["T"]
    n_new = r.multinomial(T - S, np.ones(S) / S) + 1 if T > S else np.ones(S, np.int64)
    spans, off, computed = [], [0], []
    for s in range(S):
        n = max(1, int(c["spans"] * r.uniform(0.3, 1.0)))
        k = np.zeros((n, 4), np.int64)
        k[:, 0] = r.randint(1, 60, n)                    # text
        g = np.arange(n) % 2 == 1                        # every other span an image or a frame group
        k[g, 0] = r.randint(1, 3, g.sum())
        k[g, 1] = r.randint(2, 9, g.sum())
        k[g, 2] = r.randint(2, 9, g.sum())
        k[:, 3] = r.randint(1, 5, n)
        total = int(np.where(k[:, 1] > 0, k[:, 0] * k[:, 1] * k[:, 2], k[:, 0]).sum())
        computed.append(max(0, total - int(n_new[s]) + r.randint(0, 8)))
        spans.append(k)
        off.append(off[-1] + n)
    return np.concatenate(spans).astype(np.int32), np.array(off, np.int32), np.array(computed, np.int32), n_new.astype(np.int32)


def _freqs(c):
    """Frequency (radians per position) and axis of each pair of a head."""
    half = c["D"] // 2
    j = np.arange(half)
    s = [half - 2 * (half * 3 // 8), half * 3 // 8, half * 3 // 8]
    f = 1e6 ** (-j / half)
    if c["layout"] == "sections":
        axis = np.repeat(np.arange(3), s)
    elif c["layout"] == "interleaved":
        axis = np.where((j % 3 == 1) & (j < 3 * s[1]), 1, np.where((j % 3 == 2) & (j < 3 * s[2]), 2, 0))
    else:                                                # two axes, each with all the frequencies
        a = half // 2
        axis = (j >= a).astype(np.int64)
        f = 1e4 ** (-np.where(j >= a, j - a, j) / np.where(j >= a, half - a, a))
    return f.astype(np.float64), axis.astype(np.int32)


# ---- the state of a call ----

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) % (1 << 60))


def _rows(g, T, H, Hkv, D, dt, fused):
    """q, k and v rows: of their own, or as one projection wrote them behind each other."""
    if fused:
        x = torch.randn(T, H + 2 * Hkv, D, generator=g, device="cuda").to(dt)
        return x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:]
    return tuple(torch.randn(T, n, D, generator=g, device="cuda").to(dt) for n in (H, Hkv, Hkv))


def prepare(case, seed):
    c, g = case, _gen(seed)
    dev = "cuda"
    s = {"case": c}
    if c["op"] == "attn":
        lens = _lens(c)
        qsl = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
        s["q"], s["k"], s["v"] = _rows(g, int(qsl[-1]), c["H"], c["Hkv"], c["D"], DTYPES[c["type"]], c["fused"])
        s["qsl"], s["longest"] = torch.as_tensor(qsl).to(dev), int(lens.max())
        s["row_end"] = torch.as_tensor(_row_end(c, lens)).to(dev) if c["images"] else None
        if own:
            import iian_amd as pa
            s["out"] = torch.empty(s["q"].shape, dtype=s["q"].dtype, device=dev)
            s["call"] = pa.bind_prompt_attn(
                s["q"], s["k"], s["v"], s["qsl"], s["longest"],
                pa.PagedAttnParams(scale=c["D"] ** -0.5, softcap=c["softcap"], causal=c["causal"], n_swa=c["n_swa"]),
                out=s["out"], row_end=s["row_end"])
    elif c["op"] == "rope":
        T, H, Hkv, D = c["T"], c["H"], c["Hkv"], c["D"]
        dt = DTYPES[c["type"]]
        s["q"], s["k"], s["v"] = _rows(g, T, H, Hkv, D, dt, c["fused"])
        f, axis = _freqs(c)
        s["freqs"], s["axis"] = torch.as_tensor(f).to(dev), torch.as_tensor(axis).to(dev)
        s["pos"] = torch.randint(0, c["pos_hi"], (3, T), generator=g, device=dev, dtype=torch.int32)
        s["qw"], s["kw"] = ((1 + 0.2 * torch.randn(D, generator=g, device=dev)) if c["norm"] else None for _ in range(2))
        cells = -(-(T + 100) // BS) * BS
        s["slots"] = torch.randperm(cells, generator=g, device=dev)[:T].contiguous()
        bytes_ = int(ELEM[c["pool"]] * Hkv * D)
        s["k_pool"], s["v_pool"] = (torch.zeros(cells, bytes_, dtype=torch.uint8, device=dev) for _ in range(2))
        if own:
            import iian_amd as pa
            ty = POOL_TYPES[c["pool"]]
            s["pools"] = [pa.KVPool.wrap(s[p], Hkv * D, ty) for p in ("k_pool", "v_pool")]
            s["q_out"] = torch.empty(T, H, D, dtype=dt, device=dev)
            s["call"] = pa.bind_mrope_set_rows_kv(
                s["pools"][0], s["pools"][1], s["k"], s["v"], s["slots"], s["pos"], s["freqs"], s["axis"], q=s["q"],
                q_out=s["q_out"], neox=c["neox"], q_norm=s["qw"], k_norm=s["kw"], norm_eps=EPS)
    else:
        spans, off, computed, n_new = _spans(c)
        perm = np.random.RandomState(seed % (1 << 31))     # other inputs of another seed: other texts between the grids
        text = spans[:, 1] == 0
        spans[text, 0] += perm.randint(0, 3, text.sum()).astype(np.int32)
        qsl = np.concatenate([[0], np.cumsum(n_new)]).astype(np.int32)
        for k, v in (("spans", spans), ("off", off), ("computed", computed), ("qsl", qsl)):
            s[k] = torch.as_tensor(v).to(dev)
        if own:
            import iian_amd as pa
            s["pos"] = torch.empty(3, c["T"], dtype=torch.int32, device=dev)
            s["row_end"] = torch.empty(c["T"], dtype=torch.int32, device=dev)
            s["call"] = pa.bind_mrope_positions(s["spans"], s["off"], s["computed"], s["qsl"], s["pos"],
                                                row_end=s["row_end"], grid_full=c["full"])
    return s


# ---- one pass ----

def _plain_attn(s):
    c = s["case"]
    T, H, D = s["q"].shape
    Hkv, G, L = c["Hkv"], c["H"] // c["Hkv"], s["longest"]
    start = s["qsl"][:-1].long()
    lens = s["qsl"][1:].long() - start
    i = torch.arange(L, device=s["q"].device)
    rows = (start[:, None] + i).clamp(max=T - 1)                                           # [S, L]
    q = s["q"].float()[rows].view(-1, L, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(-1, Hkv, G * L, D)
    k = s["k"].float()[rows].permute(0, 2, 3, 1)
    v = s["v"].float()[rows].permute(0, 2, 1, 3).contiguous()
    x = (q @ k.contiguous()).view(-1, Hkv, G, L, L).mul_(D ** -0.5)
    if c["softcap"]:
        x = x.div_(c["softcap"]).tanh_().mul_(c["softcap"])
    if s["row_end"] is not None:
        end = s["row_end"].long()[rows]
    else:
        end = (i + 1).expand(lens.numel(), L) if c["causal"] else lens[:, None].expand(-1, L)
    see = (i < end[:, :, None]) & (i < lens[:, None, None])
    if c["n_swa"]:
        see = see & (i[:, None] - i < c["n_swa"])
    x = x.masked_fill_(~see[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(torch.isinf(top), 0.0, top)).exp_()
    total = x.sum(-1, keepdim=True)
    o = (x.view(-1, Hkv, G * L, L) @ v).view(-1, Hkv, G, L, D) / torch.where(total == 0, 1.0, total)
    t = torch.arange(T, device=q.device)
    seq = torch.searchsorted(s["qsl"][1:].long(), t, right=True)
    o = o.permute(0, 3, 1, 2, 4).reshape(lens.numel(), L, H, D)
    return o[seq, t - start[seq]].to(s["q"].dtype)


def _plain_norm(x, w):
    x = x.float()
    return x if w is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w


def _plain_rotate(x, cos, sin, neox):
    if neox:
        a, b = x.chunk(2, -1)
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)


def _plain_q8(x):
    """Blocks of 32 values: the scale in f16, then the values as 8-bit steps of it."""
    b = x.reshape(x.shape[0], -1, 32)
    top = b.abs().amax(-1, keepdim=True)
    q = (b * torch.where(top > 0, 127.0 / top, 0.0)).round().clamp(-128, 127).to(torch.int8)
    d = (top / 127.0).to(torch.float16)
    return torch.cat([d.view(torch.uint8), q.view(torch.uint8)], -1).reshape(x.shape[0], -1)


def _plain_rope(s):
    c = s["case"]
    a = s["pos"].double()[s["axis"].long()].T * s["freqs"]                                 # [T, D/2]
    cos, sin = a.cos().float()[:, None], a.sin().float()[:, None]
    q = _plain_rotate(_plain_norm(s["q"], s["qw"]), cos, sin, c["neox"]).to(s["q"].dtype)
    k = _plain_rotate(_plain_norm(s["k"], s["kw"]), cos, sin, c["neox"]).flatten(1)
    for pool, x in ((s["k_pool"], k), (s["v_pool"], s["v"].float().flatten(1))):
        x = _plain_q8(x) if c["pool"] == "q8_0" else x.to(DTYPES[c["pool"]]).view(torch.uint8)
        pool[s["slots"]] = x
    return q


def _plain_positions(s):
    c = s["case"]
    T, dev = c["T"], s["spans"].device
    sp = s["spans"].long()
    grid = sp[:, 1] > 0
    n = torch.where(grid, sp[:, 0] * sp[:, 1] * sp[:, 2], sp[:, 0])
    adv = torch.where(grid, torch.maximum((sp[:, 0] - 1) * sp[:, 3] + 1, torch.maximum(sp[:, 1], sp[:, 2])), sp[:, 0])
    zero = torch.zeros(1, dtype=torch.long, device=dev)
    cn, ca = torch.cat([zero, n.cumsum(0)]), torch.cat([zero, adv.cumsum(0)])              # over all requests
    off = s["off"].long()
    t = torch.arange(T, device=dev)
    qsl = s["qsl"].long()
    req = torch.searchsorted(qsl[1:], t, right=True)
    r = s["computed"].long()[req] + t - qsl[req]                                           # index in the request
    first, last = off[req], off[req + 1]
    k = torch.searchsorted(cn[1:], cn[first] + r, right=True).clamp(max=sp.shape[0])
    past = k >= last                                                                       # text after the spans
    k = torch.where(past, last - 1, k)
    i = cn[first] + r - cn[k]                                                              # index in the span
    p = ca[k] - ca[first]
    h, w = sp[k, 1].clamp(min=1), sp[k, 2].clamp(min=1)
    in_grid = grid[k] & ~past
    text = torch.where(past, ca[last] - ca[first] + r - (cn[last] - cn[first]), p + i)
    axes = torch.stack([p + i // (h * w) * sp[k, 3], p + i // w % h, p + i % w])
    end = torch.where(in_grid & c["full"], cn[k + 1] - cn[first], r + 1)
    return [torch.where(in_grid, axes, text).int(), end.int()]


def _pool_values(s, own_call):
    """The pool rows as what they stand for."""
    c = s["case"]
    if c["pool"] != "q8_0":
        return [s[p].view(DTYPES[c["pool"]]) for p in ("k_pool", "v_pool")]
    if own_call:
        import iian_amd as pa
        return [pa.dequant_q8_0(p, s["slots"]).half() for p in s["pools"]]
    got = []
    for p in ("k_pool", "v_pool"):
        b = s[p][s["slots"]].view(c["T"], -1, 34)
        got.append((b[..., :2].contiguous().view(torch.float16).float() * b[..., 2:].contiguous().view(torch.int8).float())
                   .flatten(1).half())
    return got


def run(state):
    s, op = state, state["case"]["op"]
    if own:
        s["call"]()
        if op == "attn":
            return s["out"]
        if op == "positions":
            return [s["pos"], s["row_end"]]
        return [s["q_out"], *_pool_values(s, True)]
    if op == "attn":
        return _plain_attn(s)
    if op == "positions":
        return _plain_positions(s)
    return [_plain_rope(s), *_pool_values(s, False)]


def work(case):
    c = case
    if c["op"] == "attn":
        lens = _lens(c)
        ends = _row_end(c, lens) if c["images"] else None
        T = int(lens.sum())
        return {"bytes": T * c["D"] * (2 * c["H"] + 2 * c["Hkv"]) * ELEM[c["type"]] + (4 * T if c["images"] else 0),
                "flops": 4.0 * c["H"] * c["D"] * _visible(c, lens, ends)}
    if c["op"] == "rope":
        T, H, Hkv, D = c["T"], c["H"], c["Hkv"], c["D"]
        back = T * Hkv * D * 2 * (ELEM["q8_0"] + 2) if c["pool"] == "q8_0" else 0          # read back as values
        return {"bytes": T * D * ((2 * H + 2 * Hkv) * ELEM[c["type"]] + 2 * Hkv * ELEM[c["pool"]]) + 20 * T + back,
                "flops": 0}
    spans, off, _, _ = _spans(c)
    return {"bytes": 16 * c["T"] + spans.nbytes + 12 * c["S"], "flops": 0}


# ---- the definition in 64 bits ----

def _exact_attn(c, s):
    lens = _lens(c)
    o, out = 0, []
    G = c["H"] // c["Hkv"]
    for n in (int(v) for v in lens):
        i = torch.arange(n, device="cuda")
        end = (s["row_end"][o:o + n].long() if s["row_end"] is not None else i + 1 if c["causal"] else torch.full_like(i, n))
        hide = i[None, :] >= end[:, None]
        if c["n_swa"]:
            hide |= i[:, None] - i[None, :] >= c["n_swa"]
        heads = []
        for h in range(c["H"]):
            q, k, v = (s[x][o:o + n, y].double() for x, y in (("q", h), ("k", h // G), ("v", h // G)))
            z = q @ k.T.contiguous() / math.sqrt(c["D"])
            if c["softcap"]:
                z = c["softcap"] * torch.tanh(z / c["softcap"])
            z[hide] = -math.inf
            p = torch.exp(z - z.max(1, keepdim=True).values.clamp(min=-1e300))
            total = p.sum(1, keepdim=True)
            heads.append(p @ v / torch.where(total > 0, total, torch.ones_like(total)))
        out.append(torch.stack(heads, 1))
        o += n
    return torch.cat(out)


def _exact_rope(c, s):
    angle = torch.stack([s["pos"][int(a)].double() * float(f) for a, f in zip(s["axis"].tolist(), s["freqs"].tolist())], 1)
    z = torch.polar(torch.ones_like(angle), angle)[:, None, :]                              # e^(i angle)
    half = c["D"] // 2

    def turned(x, w):
        x = x.double()
        if w is not None:
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / c["D"] + EPS) * w.double()
        pair = torch.complex(x[..., :half], x[..., half:]) if c["neox"] else torch.view_as_complex(x.view(*x.shape[:-1], half, 2).contiguous())
        pair = pair * z
        return torch.cat([pair.real, pair.imag], -1) if c["neox"] else torch.view_as_real(pair).flatten(-2)

    q, k, v = turned(s["q"], s["qw"]), turned(s["k"], s["kw"]).flatten(1), s["v"].double().flatten(1)
    if c["pool"] == "q8_0":                                # steps of 8 bits: no value between them to be compared with
        return [q, None, None]
    pools = []
    for p, x in (("k_pool", k), ("v_pool", v)):
        full = torch.zeros(s[p].shape[0], x.shape[1], dtype=torch.float64, device="cuda")
        full[s["slots"]] = x
        pools.append(full)
    return [q, *pools]


def exact(case, seed):
    if case["op"] == "positions":
        return None                                        # whole numbers
    s = prepare(case, seed)
    return _exact_attn(case, s) if case["op"] == "attn" else _exact_rope(case, s)
