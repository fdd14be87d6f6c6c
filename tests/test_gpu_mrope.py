"""Multi-axis positions and the rotary K/V write (iian_pa_mrope_positions,
iian_pa_mrope_kv_write) against plain 64-bit formulas.

Tolerance of a rotated value, relative to its pair's magnitude m (after the norm
and mscale): cos and sin 2^-24 of argument rounding, 3e-8 of the Taylor sums and
2^-24 of their last sums each (1.5e-7 together); mscale, two products and a sum, 4 * 2^-24;
with a norm the mean's sum of at most 24 rounded steps (half of it under the root), the
root, the division and two products, 16 * 2^-24 more.  Together below
1.5e-7 + 20 * 6e-8 = 1.4e-6 of m.  Rounding to 16 bits adds half a step."""
import numpy as np
import pytest
import torch

F32, F16, Q8_0 = 0, 1, 8
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def test_plain_positions_by_hand():
    """The tests' own walk over the runs, on a request small enough to write down."""
    p, e = walk([(2, 0, 0, 1), (2, 2, 3, 2), (1, 0, 0, 1)], 15, True)
    assert p[0].tolist() == [0, 1] + [2] * 6 + [4] * 6 + [5]     # the grid advances by max((2-1)*2+1, 2, 3) = 3
    assert p[1].tolist() == [0, 1] + [2, 2, 2, 3, 3, 3] * 2 + [5]
    assert p[2].tolist() == [0, 1] + [2, 3, 4] * 4 + [5]
    assert e.tolist() == [1, 2] + [14] * 12 + [15]
    p, e = walk([(1, 0, 0, 1)], 4, False)
    assert p.tolist() == [[0, 1, 2, 3]] * 3 and e.tolist() == [1, 2, 3, 4]


def walk(runs, n, full):
    """Positions and ends of a request's first n tokens."""
    pos, end, p = [], [], 0
    for t, h, w, step in runs:
        first = len(pos)
        if h == 0 and w == 0:
            pos += [(p + i,) * 3 for i in range(t)]
            end += [first + i + 1 for i in range(t)]
            p += t
        elif t > 0:
            pos += [(p + it * step, p + ih, p + iw) for it in range(t) for ih in range(h) for iw in range(w)]
            m = t * h * w
            end += [first + m] * m if full else [first + i + 1 for i in range(m)]
            p += max((t - 1) * step + 1, h, w)
    while len(pos) < n:
        pos.append((p,) * 3)
        end.append(len(pos))
        p += 1
    return np.array(pos, np.int64).reshape(-1, 3).T[:, :n], np.array(end, np.int64)[:n]


@pytest.fixture(scope="module")
def pa():
    assert torch.cuda.is_available(), "GPU tests need an MI355X"
    import iian_amd
    iian_amd._lib.load()
    return iian_amd


def cu(a, dt):
    return torch.as_tensor(np.asarray(a)).to(dt).cuda()


def run_positions(pa, runs, computed, n_new, full, T=None, row_end=True):
    off = np.concatenate([[0], np.cumsum([len(r) for r in runs])])
    flat = np.array([x for r in runs for x in r], np.int32).reshape(-1, 4)
    qsl = np.concatenate([[0], np.cumsum(n_new)])
    T = int(qsl[-1]) if T is None else T
    pos = torch.full((3, T), -7, dtype=torch.int32, device="cuda")
    end = torch.full((T,), -7, dtype=torch.int32, device="cuda") if row_end else None
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    pa.mrope_positions(cu(flat, torch.int32), cu(off, torch.int32), cu(computed, torch.int32), cu(qsl, torch.int32),
                       pos, row_end=end, grid_full=full, err_flag=err)
    return pos.cpu().numpy(), None if end is None else end.cpu().numpy(), int(err.item())


def random_runs(rng, n):
    out = []
    for _ in range(n):
        if rng.random() < 0.5:
            out.append((int(rng.integers(0, 40)), 0, 0, 1))
        else:
            out.append((int(rng.integers(0, 4)), int(rng.integers(1, 9)), int(rng.integers(1, 9)), int(rng.integers(1, 6))))
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("n_runs,new_hi,full", [
    ((0, 1, 3), 40, True), ((1,), 1, False), ((7, 12, 0, 5, 1), 300, True), ((2047, 2048, 2049), 3000, True),
    ((5000, 2), 60000, False), ((4100,) * 2, 1, True), ((3,) * 70, 9, True),
])
def test_positions(pa, n_runs, new_hi, full):
    print(f"\n[gpu] positions runs={n_runs[:4]} new<={new_hi} full={full}", flush=True)
    rng = np.random.default_rng(sum(n_runs) + new_hi)
    runs = [random_runs(rng, n) for n in n_runs]
    totals = [sum(t * max(h, 1) * max(w, 1) for t, h, w, _ in r) for r in runs]
    n_new = [int(rng.integers(0, new_hi + 1)) for _ in runs]
    computed = [int(rng.integers(0, max(1, total + 4))) if rng.random() < 0.7 else 0 for total in totals]
    pos, end, err = run_positions(pa, runs, computed, n_new, full)
    assert err == 0
    o = 0
    for r, c, n in zip(runs, computed, n_new):
        want, we = walk(r, c + n, full)
        assert np.array_equal(pos[:, o:o + n], want[:, c:])
        assert np.array_equal(end[o:o + n], we[c:])
        o += n


@pytest.mark.gpu
def test_positions_rows_past_the_last_request_and_no_row_end(pa):
    pos, end, err = run_positions(pa, [[(3, 0, 0, 1)]], [0], [3], True, T=9)
    assert err == 0 and pos[:, :3].tolist() == [[0, 1, 2]] * 3 and (pos[:, 3:] == -7).all() and (end[3:] == -7).all()
    pos, end, err = run_positions(pa, [[(1, 2, 2, 1)]], [1], [4], True, row_end=False)
    assert err == 0 and end is None and pos.tolist() == [[0, 0, 0, 2], [0, 1, 1, 2], [1, 0, 1, 2]]


@pytest.mark.gpu
@pytest.mark.parametrize("runs,computed,ok", [
    ([(-1, 0, 0, 1), (2, 0, 0, 1)], 0, [0, 1, 2]),              # a negative run counts no tokens
    ([(1, 3, 0, 1), (2, 0, 0, 1)], 0, [0, 1, 2]),               # half a grid
    ([(2, 1, 1, 0)], 0, [0, 1, 2]),                             # a step of 0 counts as 1
    ([(3, 0, 0, 1)], -2, [0, 1, 2]),
    ([(1 << 30, 0, 0, 1), (1 << 30, 0, 0, 1)], 2147483645, [2147483645, 2147483646, 2147483647]),
    ([(65536, 65536, 65536, 1)], 0, None),
])
def test_positions_flags(pa, runs, computed, ok):
    pos, end, err = run_positions(pa, [runs], [computed], [3], False)
    assert err == 8
    if ok:
        assert pos[0].tolist() == ok


@pytest.mark.gpu
def test_positions_bad_offsets(pa):
    """Offsets outside the runs, or out of order, are held inside: flagged, and no run read past the array."""
    spans, pos = cu([[2, 0, 0, 1]] * 2, torch.int32), torch.zeros(3, 4, dtype=torch.int32, device="cuda")
    for off in ([-5, 1, 2], [0, 1, 900], [0, 2, 1]):
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        pa.mrope_positions(spans, cu(off, torch.int32), cu([0, 0], torch.int32), cu([0, 2, 4], torch.int32), pos,
                           err_flag=err)
        assert int(err.item()) == 8 and pos.tolist() == [[0, 1, 0, 1]] * 3


# ---- the rotary write ----

def rotated(x, w, eps, pos, freqs, axis, neox, mscale):
    """64-bit rotated rows of x [T, heads, D], and each value's pair magnitude."""
    x = x.double().cpu().numpy()
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * w.double().cpu().numpy()
    n = 2 * len(freqs)
    a = pos.cpu().numpy().astype(np.float64)[axis].T * freqs            # [T, n/2]
    c, s = np.cos(a)[:, None] * mscale, np.sin(a)[:, None] * mscale
    i0 = np.arange(n // 2) if neox else 2 * np.arange(n // 2)
    i1 = i0 + (n // 2 if neox else 1)
    y, m = x.copy(), np.abs(x)
    x0, x1 = x[..., i0], x[..., i1]
    y[..., i0], y[..., i1] = x0 * c - x1 * s, x0 * s + x1 * c
    m[..., i0] = m[..., i1] = np.hypot(x0, x1) * max(1.0, abs(mscale))
    return y, m


def check(got, want, mag, kind):
    got = got.double().cpu().numpy().reshape(want.shape)
    tol = 1.4e-6 * mag + HALF_STEP[kind] * np.abs(want) * 1.01 + (2.0 ** -25 if kind == "f16" else 1e-30)
    bad = np.abs(got - want) > tol
    assert not bad.any(), (np.argwhere(bad)[:3], got[bad][:3], want[bad][:3])


def check_pool(pool, type_, slots, want, mag, oracle_rows=None):
    """Rows at the slots hold `want` [T, Hkv, D] as the pool's type does, all other rows the fill."""
    raw = pool.data.cpu().numpy()
    rest = np.setdiff1d(np.arange(raw.shape[0]), slots)
    assert (raw[rest] == 0x5a).all()
    rows = raw[slots]
    if type_ == Q8_0:
        b = rows.reshape(len(slots), -1, 34)
        d = b[..., :2].copy().view(np.float16).astype(np.float64)
        val = (d * b[..., 2:].view(np.int8)).reshape(want.shape)
        top = np.abs(want).reshape(len(slots), -1, 32).max(-1, keepdims=True)
        # half a step of 1/127 of the block's largest, the scale's own f16 rounding at the full range
        tol = (top / 127 * 0.5 * 1.001 + top * 2.0 ** -11 + 2.0 ** -17 + 0 * d).repeat(32, -1).reshape(want.shape) + 1.4e-6 * mag
        assert (np.abs(val - want) <= tol).all()
        return
    t = torch.as_tensor(rows.copy()).view(torch.float16 if type_ == F16 else torch.float32)
    check(t, want.reshape(len(slots), -1), mag.reshape(len(slots), -1), "f16" if type_ == F16 else "f32")


def shifted(x, by):
    """x on the GPU, `by` elements past a 16-byte boundary."""
    buf = torch.empty(x.numel() + 16, dtype=x.dtype, device="cuda")
    t = buf[by:by + x.numel()].view(x.shape)
    t.copy_(x)
    return t


def one_write(pa, T, H, Hkv, D, kind="bf16", pools=(F16, F16), Dv=None, n_dims=None, neox=True, norm=(True, True),
              fused=False, off=0, with_q=True, with_kout=True, in_place=False, mscale=1.0, far=False, n_axes=3, seed=0):
    print(f"\n[gpu] mrope T={T} H={H} Hkv={Hkv} D={D} Dv={Dv} {kind} pools={pools} n={n_dims} neox={neox} norm={norm} "
          f"fused={fused} off={off} q={with_q} kout={with_kout} in_place={in_place}", flush=True)
    g = torch.Generator().manual_seed(seed + T + D)
    Dv, n_dims, dt = Dv or D, n_dims or D, DT[kind]
    if fused:
        x = shifted(torch.randn(T, (H + Hkv) * D + Hkv * Dv, generator=g).to(dt), off)
        q = x[:, :H * D].view(T, H, D)
        k = x[:, H * D:(H + Hkv) * D].view(T, Hkv, D)
        v = x[:, (H + Hkv) * D:].view(T, Hkv, Dv)
    else:
        q, k, v = (shifted(torch.randn(T, h, d, generator=g).to(dt), off) for h, d in ((H, D), (Hkv, D), (Hkv, Dv)))
    half = n_dims // 2
    fr = 1e6 ** (-np.arange(half) / half)
    axis = np.asarray(torch.randint(0, n_axes, (half,), generator=g))
    pos = torch.randint(-10 if far else 0, 2147483647 if far else 40000, (n_axes, T), generator=g, dtype=torch.int32).cuda()
    if far:
        # the 64-bit reference's own angle is pos * freq with 2^-53 of it: keep that below 1e-9
        fr = fr * 1e-3
    qw, kw = ((1 + 0.3 * torch.randn(D, generator=g)).cuda() if on else None for on in norm)
    cells = 2 * T + 5
    slots = torch.randperm(cells, generator=g)[:T].contiguous()
    rb = {F32: 4.0, F16: 2.0, Q8_0: 34 / 32}
    kp = vp = None
    if pools:
        kp, vp = (pa.KVPool.wrap(torch.full((cells, int(rb[t] * Hkv * d)), 0x5a, dtype=torch.uint8, device="cuda"),
                                 Hkv * d, t) for t, d in zip(pools, (D, Dv)))
    want_q, mag_q = rotated(q, qw, 1e-5, pos, fr, axis, neox, mscale)
    want_k, mag_k = rotated(k, kw, 1e-5, pos, fr, axis, neox, mscale)
    want_v = v.double().cpu().numpy()
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    q_out = (q if in_place else torch.empty(T, H, D, dtype=dt, device="cuda")) if with_q else None
    k_out = (k if in_place else torch.empty(T, Hkv, D, dtype=dt, device="cuda")) if with_kout else None
    pa.mrope_set_rows_kv(kp, vp, k, v if pools else None, slots.cuda() if pools else None, pos, cu(fr, torch.float64),
                         cu(axis, torch.int32), q=q if with_q else None, q_out=q_out, k_out=k_out, neox=neox, q_norm=qw,
                         k_norm=kw, norm_eps=1e-5, mscale=mscale, err_flag=err)
    assert int(err.item()) == 0
    if with_q:
        check(q_out, want_q, mag_q, kind)
    if with_kout:
        check(k_out, want_k, mag_k, kind)
    if pools:
        check_pool(kp, pools[0], slots.numpy(), want_k, mag_k)
        check_pool(vp, pools[1], slots.numpy(), want_v, 0 * want_v)
    return dict(kp=kp, vp=vp, k_out=k_out, q_out=q_out, slots=slots, v=v)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [
    dict(T=1, H=32, Hkv=8, D=128), dict(T=64, H=32, Hkv=8, D=128, kind="f32", norm=(False, False)),
    dict(T=3, H=14, Hkv=2, D=64, kind="f16", pools=(Q8_0, Q8_0)), dict(T=500, H=28, Hkv=4, D=128, fused=True),
    dict(T=9000, H=2, Hkv=1, D=64, kind="f16"), dict(T=33, H=16, Hkv=8, D=256, kind="f32", pools=(F32, F32), neox=False),
    dict(T=65, H=16, Hkv=16, D=80, pools=None), dict(T=65, H=9, Hkv=3, D=72, kind="f32", fused=True, pools=(F16, F32)),
    dict(T=65, H=9, Hkv=3, D=72, fused=True),                      # 72 = 9 pieces of 8: half a piece, the row form
    dict(T=40, H=5, Hkv=5, D=96, kind="f32", pools=(Q8_0, F16)),   # Q8_0 blocks straddle the halves
    dict(T=17, H=4, Hkv=4, D=96, pools=(F16, F32), neox=False), dict(T=31, H=8, Hkv=1, D=512, kind="f16", pools=(Q8_0, F32)),
    dict(T=8, H=3, Hkv=3, D=1024, n_dims=512), dict(T=50, H=8, Hkv=2, D=128, n_dims=64, neox=False),
    dict(T=50, H=8, Hkv=2, D=128, n_dims=2, n_axes=1), dict(T=23, H=6, Hkv=2, D=33, n_dims=32, kind="f32", pools=(F32, F16)),
    dict(T=23, H=6, Hkv=2, D=2),
    dict(T=29, H=8, Hkv=2, D=128, Dv=64, pools=(Q8_0, Q8_0)), dict(T=29, H=8, Hkv=2, D=64, Dv=50, kind="f32"),
    dict(T=130, H=8, Hkv=2, D=128, off=1), dict(T=130, H=8, Hkv=2, D=128, kind="f32", off=3, fused=True),
    dict(T=70, H=8, Hkv=2, D=128, in_place=True), dict(T=70, H=8, Hkv=2, D=128, in_place=True, fused=True, off=1),
    dict(T=70, H=8, Hkv=2, D=128, with_q=False), dict(T=70, H=8, Hkv=2, D=128, with_kout=False),
    dict(T=70, H=8, Hkv=2, D=128, norm=(True, False)), dict(T=70, H=8, Hkv=2, D=80, norm=(False, True), neox=False),
    dict(T=70, H=8, Hkv=2, D=128, mscale=1.37, kind="f32"), dict(T=300, H=2, Hkv=1, D=128, far=True, kind="f32"),
    dict(T=300, H=2, Hkv=1, D=66, far=True, kind="f32", n_axes=4),
], ids=lambda k: "-".join(f"{a}{b}" for a, b in k.items()))
def test_mrope_write(pa, kw):
    one_write(pa, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("D,pools", [(128, (Q8_0, F16)), (64, (F16, Q8_0)), (96, (Q8_0, Q8_0)), (256, (F32, Q8_0))])
def test_pools_hold_the_rotated_rows_bit_for_bit(pa, oracle, D, pools):
    """With f32 rows k_out is what goes into the pool: converted as the KV write converts it."""
    r = one_write(pa, 37, 8, 4, D, kind="f32", pools=pools)
    for pool, rows, t in ((r["kp"], r["k_out"], pools[0]), (r["vp"], r["v"], pools[1])):
        want = np.full(tuple(pool.data.shape), 0x5a, np.uint8)
        assert oracle.set_rows(want, rows.cpu().numpy().reshape(37, -1), r["slots"].numpy(), t) == 0
        assert np.array_equal(pool.data.cpu().numpy(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [128, 33])
def test_bad_slots_are_skipped_and_flagged(pa, D):
    T, Hkv = 6, 2
    k = torch.randn(T, Hkv, D, device="cuda")
    kp, vp = (pa.KVPool.wrap(torch.full((8, 4 * Hkv * D), 0x5a, dtype=torch.uint8, device="cuda"), Hkv * D, F32) for _ in range(2))
    slots = torch.tensor([0, -1, 8, 1 << 40, 7, 3], device="cuda")
    fr, ax = torch.ones(16, dtype=torch.float64, device="cuda"), torch.zeros(16, dtype=torch.int32, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    ko = torch.empty_like(k)
    pa.mrope_set_rows_kv(kp, vp, k, k, slots, torch.zeros(1, T, dtype=torch.int32, device="cuda"), fr, ax, k_out=ko, err_flag=err)
    assert int(err.item()) == 1 and torch.equal(ko, k)          # position 0 turns nothing
    rows = kp.data.view(torch.float32)
    assert all(torch.equal(rows[s], k[t].flatten()) for t, s in ((0, 0), (4, 7), (5, 3)))
    assert (kp.data[[1, 2, 4, 5, 6]] == 0x5a).all() and (vp.data[[1, 2, 4, 5, 6]] == 0x5a).all()


@pytest.mark.gpu
def test_an_axis_outside_is_held_inside(pa):
    k = torch.randn(3, 1, 64, device="cuda")
    pos = torch.tensor([[1, 2, 3], [40, 50, 60]], dtype=torch.int32, device="cuda")
    fr = torch.ones(32, dtype=torch.float64, device="cuda")
    a, b = torch.empty_like(k), torch.empty_like(k)
    pa.mrope_set_rows_kv(None, None, k, None, None, pos, fr, cu([-3] * 16 + [7] * 16, torch.int32), k_out=a)
    pa.mrope_set_rows_kv(None, None, k, None, None, pos, fr, cu([0] * 16 + [1] * 16, torch.int32), k_out=b)
    assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 66])
def test_negative_frequencies_turn_back(pa, D):
    """Rotated by a table and then by its negative, a row is itself again; tiny frequencies of either sign turn nothing."""
    T = 50
    k = torch.randn(T, 2, D, device="cuda")
    pos = torch.randint(-4000, 1000000, (1, T), dtype=torch.int32, device="cuda")
    fr = 1e4 ** (-torch.arange(D // 2, dtype=torch.float64, device="cuda") / (D // 2))
    ax = torch.zeros(D // 2, dtype=torch.int32, device="cuda")
    a, b = torch.empty_like(k), torch.empty_like(k)
    pa.mrope_set_rows_kv(None, None, k, None, None, pos, fr, ax, k_out=a)
    pa.mrope_set_rows_kv(None, None, a, None, None, pos, -fr, ax, k_out=b)
    pair = (k[..., :D // 2] ** 2 + k[..., D // 2:] ** 2).sqrt().repeat(1, 1, 2)
    assert ((b - k).abs() <= 2.8e-6 * pair).all()
    pos.fill_(2147483647)
    for tiny in (1e-18, -1e-18, -1e-300):
        pa.mrope_set_rows_kv(None, None, k, None, None, pos, 0 * fr + tiny, ax, k_out=a)
        assert ((a - k).abs() <= 1.4e-6 * pair).all()


@pytest.mark.gpu
def test_one_axis_agrees_with_the_rope_write(pa):
    """All axes at the token's index: the rotation iian_pa_rope_kv_write makes, whose chained fp32 angle is off by
    up to (j + 1) roundings of 2^-24 at pair j: at position p < 64, 64 * p * 2^-24 < 2.5e-4 of the pair."""
    T, H, Hkv, D = 40, 8, 2, 128
    q, k, v = (torch.randn(T, h, D, device="cuda") for h in (H, Hkv, Hkv))
    slots = torch.arange(T, device="cuda")
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    rope = pa.RopeParams(n_dims=D, mode=2, freq_base=1e6)
    pools = [pa.KVPool(T, Hkv * D, F32) for _ in range(4)]
    want = pa.rope_set_rows_kv(pools[0], pools[1], k.view(T, -1), v.view(T, -1), slots, pos, rope, Hkv, q=q)
    fr, ax, ms = pa.mrope_frequencies(rope, (16, 24, 24))
    got = pa.mrope_set_rows_kv(pools[2], pools[3], k, v, slots, pos.expand(3, T).contiguous(), fr, ax, q=q, mscale=ms)
    assert (got - want).abs().max() < 2.5e-4 * q.abs().max() * 1.5
    assert torch.equal(pools[1].data, pools[3].data)


@pytest.mark.gpu
def test_refusals(pa):
    k = torch.randn(4, 2, 64, device="cuda")
    pos = torch.zeros(3, 4, dtype=torch.int32, device="cuda")
    fr, ax = torch.ones(32, dtype=torch.float64, device="cuda"), torch.zeros(32, dtype=torch.int32, device="cuda")
    call = lambda **kw: pa.mrope_set_rows_kv(**{**dict(k_pool=None, v_pool=None, k_rows=k, v_rows=None, slots=None, pos=pos,
                                                     freqs=fr, axis=ax, k_out=torch.empty_like(k)), **kw})
    call()
    for bad in (dict(k_out=None), dict(pos=pos[:, :3]), dict(pos=pos.long()), dict(freqs=fr.float()), dict(axis=ax[:3]),
                dict(k_rows=k.transpose(1, 2)), dict(k_rows=k.double()), dict(slots=torch.arange(4, device="cuda")),
                dict(q=k.half(), q_out=k.half()), dict(q_out=k), dict(k_norm=torch.ones(63, device="cuda")),
                dict(k_rows=k.cpu()), dict(k_pool=pa.KVPool(8, 128, F16)), dict(q=k, q_out=torch.empty(4, 2, 32, device="cuda"))):
        with pytest.raises(ValueError):
            call(**bad)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [128, 66])
def test_offsets_past_32_bits(pa, D):
    """Pool rows past 2^32 elements, and tokens far apart."""
    T, Hkv = 70, 8
    cells = (1 << 32) // (Hkv * D) + 4000
    pool = torch.empty(cells, 2 * Hkv * D, dtype=torch.uint8, device="cuda")
    kp, vp = pa.KVPool.wrap(pool, Hkv * D, F16), pa.KVPool(cells, Hkv, F16)
    rows = torch.empty(T, (1 << 26) + 64, dtype=torch.float16, device="cuda")[:, :Hkv * D].view(T, Hkv, D)
    rows.copy_(torch.randn(T, Hkv, D))
    v = torch.randn(T, Hkv, 1, device="cuda").half()
    slots = torch.arange(cells - T, cells, device="cuda")
    pos = torch.randint(0, 9999, (2, T), dtype=torch.int32, device="cuda")
    fr = torch.rand(D // 2, dtype=torch.float64, device="cuda")
    ax = torch.randint(0, 2, (D // 2,), dtype=torch.int32, device="cuda")
    ko = torch.empty(T, Hkv, D, dtype=torch.float16, device="cuda")
    pa.mrope_set_rows_kv(kp, vp, rows, v, slots, pos, fr, ax, k_out=ko)
    want, mag = rotated(rows, None, 0, pos, fr.cpu().numpy(), ax.cpu().numpy().astype(int), True, 1.0)
    check(ko, want, mag, "f16")
    assert torch.equal(kp.view_f16()[cells - T:], ko.view(T, -1))
    assert torch.equal(vp.view_f16()[cells - T:], v.view(T, -1))


@pytest.mark.gpu
def test_streams_and_graphs(pa):
    """Positions and the write captured together, replayed with new inputs between eager work, and on two streams at once."""
    T, H, Hkv, D = 60, 8, 2, 128
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(T, h, D, generator=g).bfloat16().cuda() for h in (H, Hkv, Hkv))
    spans = cu([[9, 0, 0, 1], [2, 3, 4, 1], [7, 0, 0, 1]], torch.int32)
    off, qsl = cu([0, 3], torch.int32), cu([0, T], torch.int32)
    fr, ax, ms = pa.mrope_frequencies(pa.RopeParams(n_dims=D, freq_base=1e6), (16, 24, 24))
    slots = torch.randperm(T + 4, generator=g)[:T].cuda()

    def step(computed):
        pos = torch.empty(3, T, dtype=torch.int32, device="cuda")
        kp, vp = pa.KVPool(T + 4, Hkv * D, F16), pa.KVPool(T + 4, Hkv * D, F16)
        qo = torch.empty_like(q)
        return pos, kp, vp, qo, computed

    def run(s):
        pa.mrope_positions(spans, off, s[4], qsl, s[0])
        pa.mrope_set_rows_kv(s[1], s[2], k, v, slots, s[0], fr, ax, q=q, q_out=s[3], mscale=ms)

    computed = cu([5], torch.int32)
    eager, captured = step(computed), step(computed)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(captured)
    for n in (0, 3, 900):
        computed.fill_(n)
        run(eager)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(eager[0], captured[0]) and torch.equal(eager[3], captured[3])
        assert torch.equal(eager[1].data, captured[1].data) and torch.equal(eager[2].data, captured[2].data)
        captured[3].zero_()
    both = [step(computed), step(computed)]
    torch.cuda.synchronize()
    for s in both:
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                run(s)
    torch.cuda.synchronize()
    assert all(torch.equal(s[3], eager[3]) and torch.equal(s[1].data, eager[1].data) for s in both)
