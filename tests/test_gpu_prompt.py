"""Attention over whole prompts (iian_pa_prompt_attention) against its definition in 64 bits.

Tolerance of an output value, with A = sum_j p_j |v_j|, B = sum_j |v_j| over the visible tokens, Q = scale * max_j
sum_d |q_d k_jd|, u half a step of the type (bf16 2^-8, f16 2^-11, f32 0) and e = 2^-24:
  scores: fp32 sums of D exact products, D e Q, twice that for rounded partial scales (a softcap only shrinks it); for f32 rows
  the pairs of f16 terms leave 2^-21 of each product, 2^-21 Q.  A score's error is p's relative error, and
  the sum's: 2 (2 D e + 2^-21 [f32]) Q A.
  probabilities: u (to the type) or 2^-21 (f32 rows: p's and v's pairs, and the product of the rests left out), and f16's smallest
  step, 2^-25 for each token (the largest p is 1 or more): (u + 2^-21 [f32]) A + 2^-25 B.  The sum of p is taken before or after this
  rounding: again u A.
  fp32 sums over N tokens: 2 N e A, exponentials and the division 16 e A.
  The result's own rounding: u |out|, and f16's smallest step 2^-25."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


@pytest.fixture(scope="module")
def pa():
    assert torch.cuda.is_available(), "GPU tests need an MI355X"
    import iian_amd
    iian_amd._lib.load()
    return iian_amd


def definition(q, k, v, lens, scale, softcap=0.0, causal=True, n_swa=0, row_end=None):
    """(out, A, B, Q, N) in 64 bits on the CPU; a hidden token's k and v are not read."""
    q, k, v = (x.double().cpu() for x in (q, k, v))
    H, G = q.shape[1], q.shape[1] // k.shape[1]
    outs = []
    o = 0
    for n in lens:
        i = torch.arange(n)
        end = row_end[o:o + n].long().cpu().clamp(0, n) if row_end is not None else i + 1 if causal else torch.full((n,), n)
        see = i < end[:, None]
        if n_swa:
            see &= i[:, None] - i < n_swa
        for h in range(H if n else 0):
            qq, kk, vv = q[o:o + n, h], k[o:o + n, h // G], v[o:o + n, h // G]
            x = scale * (qq @ kk.T)
            big = abs(scale) * (qq.abs() @ kk.abs().T)
            if softcap:
                x = softcap * torch.tanh(x / softcap)
            x = torch.where(see, x, -torch.inf)
            p = torch.exp(x - x.amax(1, keepdim=True).clamp(min=-1e300))
            p = torch.where(see, p, 0.0)
            tot = p.sum(1, keepdim=True)
            p = p / torch.where(tot > 0, tot, 1.0)
            any_v = torch.where(torch.isfinite(vv), vv, 0.0)
            outs.append((o, h, p @ any_v, p @ any_v.abs(), see.double() @ any_v.abs(),
                         torch.where(see & torch.isfinite(big), big, 0.0).amax(1)))
        o += n
    T, Dv = q.shape[0], v.shape[2]
    out, A, B = (torch.zeros(T, H, Dv, dtype=torch.float64) for _ in range(3))
    Q = torch.zeros(T, H, 1, dtype=torch.float64)
    for o, h, y, a, b, s in outs:
        n = y.shape[0]
        out[o:o + n, h], A[o:o + n, h], B[o:o + n, h], Q[o:o + n, h, 0] = y, a, b, s
    return out, A, B, Q, max(list(lens) + [1])


def tolerance(kind, D, out, A, B, Q, N):
    u, e, f32 = U[kind], 2.0 ** -24, 2.0 ** -21 if kind == "f32" else 0.0
    return (2 * (2 * D * e + f32) * Q * A + (2 * u + f32 + 2 * N * e + 16 * e) * A + 2.0 ** -25 * B + u * out.abs()
            + (2.0 ** -25 if kind == "f16" else 1e-30))


def rows(g, T, H, Hkv, D, Dv, kind, fused=False, off=0, mult=1.0):
    dt = DT[kind]
    sizes = (H * D, Hkv * D, Hkv * Dv)
    if fused:
        buf = torch.empty(T * sum(sizes) + 16, dtype=dt, device="cuda")
        x = buf[off:off + T * sum(sizes)].view(T, sum(sizes))
        x.copy_(torch.randn(T, sum(sizes), generator=g) * mult)
        q, k, v = x.split(sizes, 1)
    else:
        q, k, v = (torch.empty(T * n + 16, dtype=dt, device="cuda")[off:off + T * n].view(T, n) for n in sizes)
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g) * mult)
    return q.unflatten(1, (H, D)), k.unflatten(1, (Hkv, D)), v.unflatten(1, (Hkv, Dv))


def one(pa, lens, H, Hkv, D, kind="bf16", Dv=None, causal=True, n_swa=0, softcap=0.0, ends=None, fused=False, off=0,
        mult=1.0, scale=None, lead=0, tail=0, seed=0, change=None, max_q=None):
    """One call on prompts of these lengths, behind `lead` and before `tail` rows that belong to none."""
    print(f"\n[gpu] prompt lens={list(lens)[:6]} H={H} Hkv={Hkv} D={D} Dv={Dv} {kind} causal={causal} swa={n_swa} cap={softcap} "
          f"ends={ends} fused={fused} off={off} mult={mult}", flush=True)
    Dv = Dv or D
    g = torch.Generator().manual_seed(seed + sum(lens) + D)
    T = lead + sum(lens) + tail
    q, k, v = rows(g, T, H, Hkv, D, Dv, kind, fused, off, mult)
    for x in (q, k, v):                                          # what belongs to no prompt must not be read
        x[:lead] = x[T - tail:] = float("nan")
    qsl = (lead + np.concatenate([[0], np.cumsum(lens)])).astype(np.int32)
    row_end = None
    if ends is not None:
        row_end = torch.zeros(T, dtype=torch.int32)
        o = lead
        for n in lens:
            row_end[o:o + n] = torch.as_tensor(ends(n, g), dtype=torch.int32)
            o += n
    if change:
        change(q, k, v, lead)
    scale = D ** -0.5 if scale is None else scale
    out = torch.full((T, H, Dv), 77.0, dtype=DT[kind], device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    prm = pa.PagedAttnParams(scale=scale, softcap=softcap, causal=causal, n_swa=n_swa)
    pa.prompt_attn(q, k, v, torch.as_tensor(qsl).cuda(), max_q or max(max(lens), 1), prm, out=out,
                   row_end=None if row_end is None else row_end.cuda(), err_flag=err)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    assert (out[:lead] == 77).all() and (out[T - tail:] == 77).all()
    mid = slice(lead, T - tail)
    d = definition(q[mid], k[mid], v[mid], lens, scale, softcap, causal, n_swa,
                   None if row_end is None else row_end[mid])
    got = out[mid].double().cpu()
    over = (got - d[0]).abs() - tolerance(kind, D, *d)
    assert not torch.isnan(got).any()
    assert (over <= 0).all(), (over.max(), torch.nonzero(over > 0)[:4], (got - d[0]).abs().max())
    return q, k, v, out, qsl


def image_ends(n, g):
    e = torch.arange(1, n + 1)
    a = 5
    while a < n:
        b = min(n, a + int(torch.randint(3, 120, (1,), generator=g)))
        e[a:b] = b
        a = b + int(torch.randint(1, 60, (1,), generator=g))
    return e


ENDS = {"images": image_ends, "any": lambda n, g: torch.randint(-5, n + 9, (n,), generator=g),
        "none": lambda n, g: torch.zeros(n, dtype=torch.int64), "last_only": lambda n, g: (torch.arange(n) == n - 1) * n}


LENS = [(1,), (1, 2, 3, 1), (16,), (31, 33), (63, 64, 65), (100, 1, 0, 257), (400, 129), (0, 5, 0, 0, 40)]


@pytest.mark.parametrize("lens", LENS, ids=str)
@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads", [(8, 2, 128), (3, 3, 64)], ids=str)
def test_lengths(pa, lens, kind, heads):
    one(pa, lens, *heads, kind=kind, lead=3, tail=2)


@pytest.mark.parametrize("D,Dv", [(8, 8), (16, 64), (32, 32), (40, 24), (64, 128), (72, 72), (80, 80), (96, 96), (96, 64),
                                  (112, 112), (128, 64), (160, 160), (192, 128), (200, 256), (256, 256), (256, 8)])
@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
def test_head_sizes(pa, D, Dv, kind):
    one(pa, (70, 150), 4, 2, D, Dv=Dv, kind=kind)


MANY = [1 + 37 * i % 250 for i in range(45)]    # enough row blocks that no two waves share rows


@pytest.mark.parametrize("D,Dv", [(64, 64), (48, 8), (80, 96), (128, 128), (128, 104), (256, 256), (136, 200)])
@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
def test_many_prompts(pa, D, Dv, kind):
    one(pa, MANY, 16, 8, D, Dv=Dv, kind=kind, lead=2, tail=3)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("kw", [
    dict(causal=False), dict(n_swa=40), dict(causal=False, n_swa=70), dict(softcap=5.0), dict(scale=-0.1), dict(mult=6.0),
    dict(fused=True, off=8), dict(images=True), dict(images=True, n_swa=50), dict(empty=True),
], ids=str)
def test_many_prompts_masked(pa, kw, kind):
    ends = image_ends if kw.get("images") else ENDS["any"] if kw.get("empty") else None
    one(pa, MANY, 16, 8, 128, kind=kind, ends=ends, **{k: v for k, v in kw.items() if k not in ("images", "empty")})


@pytest.mark.parametrize("D,kind", [(64, "f16"), (80, "bf16"), (96, "f32"), (256, "bf16"), (256, "f32")])
@pytest.mark.parametrize("kw", [dict(causal=False), dict(n_swa=50, softcap=8.0), dict(images=True, n_swa=90), dict(empty=True)], ids=str)
def test_many_prompts_masked_at_other_head_sizes(pa, D, kind, kw):
    ends = image_ends if kw.get("images") else ENDS["any"] if kw.get("empty") else None
    one(pa, MANY, 16, 8, D, kind=kind, ends=ends, lead=1, **{k: v for k, v in kw.items() if k not in ("images", "empty")})


@pytest.mark.parametrize("lens,H,Hkv,D", [((1100, 3, 200), 16, 16, 128), ((700, 650), 20, 20, 96), ((1600, 40), 12, 12, 64)])
@pytest.mark.parametrize("kw", [dict(), dict(n_swa=300, softcap=8.0), dict(images=True)], ids=str)
def test_f32_longer_prompts(pa, lens, H, Hkv, D, kw):
    """Calls whose last row blocks are their critical path: 8 waves that share rows."""
    one(pa, lens, H, Hkv, D, kind="f32", ends=image_ends if kw.get("images") else None,
        **{k: v for k, v in kw.items() if k != "images"})


@pytest.mark.parametrize("D,kind", [(80, "bf16"), (256, "f16"), (256, "f32")])
def test_hidden_values_of_many_prompts(pa, D, kind):
    """As below, with row blocks of every kind of workgroup: each prompt's last token holds NaN and infinities, which the
    tokens before it do not see."""
    g = torch.Generator().manual_seed(9)
    T = sum(MANY)
    q, k, v = rows(g, T, 16, 8, D, D, kind)
    qsl = torch.tensor(np.concatenate([[0], np.cumsum(MANY)]), dtype=torch.int32, device="cuda")
    prm = pa.PagedAttnParams(scale=D ** -0.5)
    want = pa.prompt_attn(q, k, v, qsl, max(MANY), prm)
    last = qsl[1:].long() - 1
    keep = torch.ones(T, dtype=torch.bool, device="cuda")
    keep[last] = False
    for bad in (float("nan"), float("inf")):
        k[last, :, 3] = bad
        v[last, :, 5] = -bad
        v[last, 0] = bad
        assert torch.equal(pa.prompt_attn(q, k, v, qsl, max(MANY), prm)[keep], want[keep])


@pytest.mark.parametrize("S,L", [(64, 30), (65, 30), (200, 9), (1500, 3), (5000, 1)])
@pytest.mark.parametrize("causal", [True, False])
def test_prompt_counts(pa, S, L, causal):
    """The order of the row blocks: up to 64 prompts, more, and more than 64 shares of 64."""
    one(pa, [1 + (7 * i) % L for i in range(S)], 4, 4, 64, causal=causal, lead=1)


def test_one_long_prompt(pa):
    one(pa, (3000,), 8, 8, 64, kind="f16")


@pytest.mark.parametrize("D,Dv,kind", [(1, 1, "f32"), (33, 33, "bf16"), (100, 100, "f16"), (128, 33, "bf16"), (320, 320, "f16"),
                                       (576, 512, "bf16"), (1024, 1024, "f32"), (64, 257, "f32")])
def test_head_sizes_of_the_row_form(pa, D, Dv, kind):
    one(pa, (70, 3), 2, 1, D, Dv=Dv, kind=kind)


@pytest.mark.parametrize("H,Hkv", [(1, 1), (7, 1), (14, 2), (9, 3), (28, 4), (40, 8), (16, 16), (64, 2), (200, 1)])
def test_head_layouts(pa, H, Hkv):
    one(pa, (37, 90), H, Hkv, 64)


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("kw", [
    dict(causal=False), dict(n_swa=1), dict(n_swa=50), dict(n_swa=64), dict(causal=False, n_swa=70), dict(softcap=5.0),
    dict(softcap=20.0, causal=False, n_swa=33), dict(scale=0.0), dict(scale=-0.1), dict(mult=4.0), dict(mult=6.0, softcap=30.0),
    dict(mult=1e-4), dict(fused=True), dict(fused=True, off=8), dict(max_q=600),
], ids=str)
def test_masks_and_values(pa, kw, kind):
    one(pa, (300, 77, 223), 8, 2, 128, kind=kind, **kw)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("ends", list(ENDS))
@pytest.mark.parametrize("n_swa", [0, 40])
def test_row_ends(pa, ends, kind, n_swa):
    one(pa, (190, 1, 64, 333), 8, 2, 128, kind=kind, ends=ENDS[ends], n_swa=n_swa)


@pytest.mark.parametrize("off,D", [(1, 128), (4, 64), (3, 256)])
@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_unaligned_rows(pa, off, D, kind):
    one(pa, (70, 41), 4, 2, D, kind=kind, off=off, fused=off == 3)


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("what", ["nan", "inf", "big"])
@pytest.mark.parametrize("H,Hkv", [(8, 2), (64, 32)])
def test_hidden_values_reach_nothing(pa, kind, what, H, Hkv):
    """A later token's k and v, whatever they hold, leave the tokens before it alone."""
    bad = {"nan": float("nan"), "inf": float("inf"), "big": torch.finfo(DT[kind]).max}[what]

    def change(q, k, v, lead):
        for t in (40, 63, 64, 130, 199):
            k[t, :, 3] = bad
            v[t, :, 5] = bad
            v[t, 0, 9] = -bad
    # rows from 40 on see one: compared up to there, and from the next prompt on
    g = torch.Generator().manual_seed(1)
    q, k, v = rows(g, 300, H, Hkv, 128, 128, kind)
    qsl = torch.tensor([0, 200, 300], dtype=torch.int32, device="cuda")
    prm = pa.PagedAttnParams(scale=128 ** -0.5)
    clean = pa.prompt_attn(q, k, v, qsl, 200, prm).clone()
    change(q, k, v, 0)
    got = pa.prompt_attn(q, k, v, qsl, 200, prm)
    d = definition(q[:40], k[:40], v[:40], (40,), 128 ** -0.5)
    assert ((got[:40].double().cpu() - d[0]).abs() <= tolerance(kind, 128, *d)).all()
    assert torch.equal(got[200:], clean[200:])
    # a window that has left them behind
    w = pa.prompt_attn(q, k, v, qsl, 200, pa.PagedAttnParams(scale=128 ** -0.5, n_swa=20))
    d = definition(q[:200], k[:200], v[:200], (200,), 128 ** -0.5, n_swa=20)
    rows_ok = [i for i in range(200) if not any(i - 20 < t <= i for t in (40, 63, 64, 130, 199))]
    over = (w[:200].double().cpu() - d[0]).abs() - tolerance(kind, 128, *d)
    assert (over[rows_ok] <= 0).all()


@pytest.mark.parametrize("kind", ["f16", "f32"])
def test_scores_of_the_lowest_value(pa, kind):
    """K rows of the type's lowest value and of -inf against a positive q: weights of zero, and a row that sees only
    such tokens ends finite or zero."""
    q, k, v = rows(torch.Generator().manual_seed(2), 90, 4, 2, 64, 64, kind)
    q.abs_()
    k[10:20] = float("-inf")
    qsl = torch.tensor([0, 90], dtype=torch.int32, device="cuda")
    got = pa.prompt_attn(q, k, v, qsl, 90, pa.PagedAttnParams(scale=0.125))
    keep = [i for i in range(90) if not 10 <= i < 20]
    kk, vv = k.clone(), v.clone()
    d = definition(q[:10], k[:10], v[:10], (10,), 0.125)
    assert ((got[:10].double().cpu() - d[0]).abs() <= tolerance(kind, 64, *d)).all()
    if kind == "f16":                     # enters the product as it is: -inf scores weigh nothing
        full = q.double(), kk.double(), vv.double()
        x = 0.125 * torch.einsum("id,jd->ij", full[0][89:, 0].cpu(), full[1][keep, 0].cpu())
        p = torch.softmax(x, 1) @ full[2][keep, 0].cpu()
        assert ((got[89, 0].double().cpu() - p[0]).abs() < 4e-3).all()


def test_a_longer_prompt_than_declared_is_flagged(pa):
    q, k, v = rows(torch.Generator().manual_seed(3), 300, 4, 2, 64, 64, "bf16")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    qsl = torch.tensor([0, 20, 300], dtype=torch.int32, device="cuda")
    prm = pa.PagedAttnParams(scale=0.125)
    got = pa.prompt_attn(q, k, v, qsl, 40, prm, err_flag=err)
    want = pa.prompt_attn(q, k, v, qsl, 280, prm)
    assert int(err.item()) == 4 and torch.equal(got[:60], want[:60])


def test_query_start_loc_outside_the_rows(pa):
    """Starts out of order or past the tokens are held inside them."""
    q, k, v = rows(torch.Generator().manual_seed(4), 64, 2, 1, 64, 64, "bf16")
    prm = pa.PagedAttnParams(scale=0.125)
    want = pa.prompt_attn(q, k, v, torch.tensor([0, 64], dtype=torch.int32, device="cuda"), 64, prm)
    got = pa.prompt_attn(q, k, v, torch.tensor([0, 900], dtype=torch.int32, device="cuda"), 64, prm)
    assert torch.equal(got, want)
    pa.prompt_attn(q, k, v, torch.tensor([-50, 70, 3, 1 << 30], dtype=torch.int32, device="cuda"), 64, prm)
    torch.cuda.synchronize()


def test_refusals(pa):
    q = torch.zeros(4, 4, 64, device="cuda", dtype=torch.bfloat16)
    k = torch.zeros(4, 2, 64, device="cuda", dtype=torch.bfloat16)
    qsl = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    prm = pa.PagedAttnParams(scale=0.125)
    pa.prompt_attn(q, k, k, qsl, 4, prm)
    for args in ((q.double(), k, k, qsl), (q, k.half(), k, qsl), (q, k[:3], k, qsl), (q, k, k[:, :1], qsl), (q, k[..., :32], k, qsl),
                 (q, k, k, qsl.long()), (q.cpu(), k, k, qsl), (q, k.transpose(1, 2).contiguous().transpose(1, 2), k, qsl)):
        with pytest.raises(ValueError):
            pa.prompt_attn(*args, 4, prm)
    with pytest.raises(ValueError):
        pa.prompt_attn(q, k, k, qsl, 4, prm, row_end=torch.zeros(3, dtype=torch.int32, device="cuda"))
    for n in (0, 5):
        with pytest.raises(pa.PagedAttnError):
            pa.prompt_attn(q, k, k, qsl, n, prm)
    with pytest.raises(pa.PagedAttnError):
        pa.prompt_attn(q[:, :3].contiguous(), k, k, qsl, 4, prm)


def test_out_in_place_of_q(pa):
    for kind, H, n in (("bf16", 8, 300), ("f32", 64, 900)):
        q, k, v = rows(torch.Generator().manual_seed(5), n, H, H // 4, 128, 128, kind)
        qsl = torch.tensor([0, n // 3, n], dtype=torch.int32, device="cuda")
        prm = pa.PagedAttnParams(scale=128 ** -0.5)
        want = pa.prompt_attn(q, k, v, qsl, n, prm)
        pa.prompt_attn(q, k, v, qsl, n, prm, out=q)
        assert torch.equal(q, want)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_offsets_past_32_bits(pa, kind):
    """Tokens far apart: element offsets of the last ones past 2^32."""
    T, H, Hkv, D = 1100, 4, 1, 64
    stride = 4000000                     # (16-bit rows: addressed per tile; the unaligned form's addresses are 64-bit)
    dt = DT[kind]
    g = torch.Generator().manual_seed(6)
    buf = torch.empty(T * stride, dtype=dt, device="cuda")
    x = buf.view(T, stride)[:, :(H + 2 * Hkv) * D]
    x.copy_(torch.randn(T, (H + 2 * Hkv) * D, generator=g))
    q, k, v = (t.unflatten(1, (n, D)) for t, n in zip(x.split((H * D, Hkv * D, Hkv * D), 1), (H, Hkv, Hkv)))
    qsl = torch.tensor([0, 500, T], dtype=torch.int32, device="cuda")
    prm = pa.PagedAttnParams(scale=0.125)
    far = pa.prompt_attn(q, k, v, qsl, T, prm)
    assert torch.equal(far, pa.prompt_attn(q.contiguous(), k.contiguous(), v.contiguous(), qsl, T, prm))
    d = definition(q[500:], k[500:], v[500:], (T - 500,), 0.125)
    assert ((far[500:].double().cpu() - d[0]).abs() <= tolerance(kind, D, *d)).all()


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_streams_and_graphs(pa, kind):
    """Two calls at once on two streams, and a captured call replayed with new inputs between eager work."""
    prm = pa.PagedAttnParams(scale=128 ** -0.5)
    sets = []
    for n, H in ((700, 32), (90, 8)):
        q, k, v = rows(torch.Generator().manual_seed(n), n, H, H // 4, 128, 128, kind)
        qsl = torch.tensor([0, n // 2, n], dtype=torch.int32, device="cuda")
        sets.append((q, k, v, qsl, n, pa.prompt_attn(q, k, v, qsl, n, prm)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for st, (q, k, v, qsl, n, _) in zip(streams, sets):
        with torch.cuda.stream(st):
            got.append([pa.prompt_attn(q, k, v, qsl, n, prm) for _ in range(5)])
    torch.cuda.synchronize()
    for g, s in zip(got, sets):
        assert all(torch.equal(y, s[5]) for y in g)
    for q, k, v, qsl, n, want in sets:
        out = torch.zeros_like(want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            pa.prompt_attn(q, k, v, qsl, n, prm, out=out)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
            k.mul_(-1)
            want = pa.prompt_attn(q, k, v, qsl, n, prm)
            out.zero_()


def test_the_same_call_gives_the_same_bits(pa):
    q, k, v = rows(torch.Generator().manual_seed(8), 2000, 16, 4, 128, 128, "f16")
    qsl = torch.tensor([0, 3, 1200, 2000], dtype=torch.int32, device="cuda")
    prm = pa.PagedAttnParams(scale=128 ** -0.5)
    a = [pa.prompt_attn(q, k, v, qsl, 1997, prm) for _ in range(4)]
    assert all(torch.equal(a[0], x) for x in a[1:])
