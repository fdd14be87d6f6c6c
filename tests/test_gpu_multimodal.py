"""The operators of a prompt with images, together as an engine uses them: the step's metadata and positions, the rotary
write, attention over the prompts' rows, then decode steps over the pool.  Checked against 64-bit formulas from the raw rows."""
import numpy as np
import pytest
import torch

from test_gpu_mrope import rotated, walk

pytestmark = pytest.mark.gpu
F32, F16, Q8_0 = 0, 1, 8


@pytest.fixture(scope="module")
def pa():
    assert torch.cuda.is_available(), "GPU tests need an MI355X"
    import iian_amd
    iian_amd._lib.load()
    return iian_amd


def attend(q, k, v, end, scale):
    """q [n, H, D] over k, v [m, Hkv, D] in 64 bits: token i sees the first end[i]."""
    G = q.shape[1] // k.shape[1]
    x = scale * np.einsum("ihd,jhd->hij", q, k.repeat(G, 1))
    x = np.where(np.arange(k.shape[0]) < end[:, None], x, -np.inf)
    p = np.exp(x - x.max(-1, keepdims=True))
    return np.einsum("hij,jhd->ihd", p / p.sum(-1, keepdims=True), v.repeat(G, 1))


@pytest.mark.parametrize("H,Hkv,D,kind", [(8, 2, 128, "f32"), (16, 8, 64, "f32")])
@pytest.mark.parametrize("pool", [F16, F32])
def test_prompt_step_then_decodes(pa, H, Hkv, D, kind, pool):
    print(f"\n[gpu] multimodal step H={H} Hkv={Hkv} D={D} pool={pool}", flush=True)
    rng = np.random.default_rng(D)
    bs, dev = 16, "cuda"
    runs = [[(20, 0, 0, 1), (2, 6, 8, 1), (11, 0, 0, 1)], [(5, 0, 0, 1)], [(3, 0, 0, 1), (1, 7, 9, 1), (40, 0, 0, 1), (4, 2, 2, 2)]]
    lens = [sum(t * max(h, 1) * max(w, 1) for t, h, w, _ in r) for r in runs]
    S, n_dec = len(runs), 3
    blocks, nb = [], 0
    perm = rng.permutation(64)
    for n in lens:
        m = -(-(n + n_dec) // bs)
        blocks.append(perm[nb:nb + m].tolist())
        nb += m
    cells = 64 * bs
    kp, vp = pa.KVPool(cells, Hkv * D, pool), pa.KVPool(cells, Hkv * D, pool)
    rope = pa.RopeParams(n_dims=D, mode=2, freq_base=1e6)
    sec = (D // 2 - 2 * (3 * D // 16), 3 * D // 16, 3 * D // 16)
    fr, ax, ms = pa.mrope_frequencies(rope, sec)
    fh, ah = fr.cpu().numpy(), ax.cpu().numpy()
    qw, kw = (1 + 0.2 * torch.randn(D, device=dev) for _ in range(2))
    spans = torch.as_tensor([x for r in runs for x in r], dtype=torch.int32).to(dev)
    off = torch.as_tensor(np.concatenate([[0], np.cumsum([len(r) for r in runs])]), dtype=torch.int32).to(dev)
    scale = D ** -0.5
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    keys, vals = [None] * S, [None] * S
    for step in range(1 + n_dec):
        computed = [0] * S if step == 0 else [n + step - 1 for n in lens]
        new = lens if step == 0 else [1] * S
        T = sum(new)
        req = pa.RequestBlocks.pack(blocks, computed, new, device=dev)
        batch = pa.build_batch(req, T, bs, max(len(b) for b in blocks), 64, max_query_len=max(new), err_flag=err)
        pos = torch.empty(3, T, dtype=torch.int32, device=dev)
        row_end = torch.empty(T, dtype=torch.int32, device=dev)
        pa.mrope_positions(spans, off, req.num_computed, batch.query_start_loc, pos, row_end=row_end, grid_full=True, err_flag=err)
        x = torch.randn(T, H + 2 * Hkv, D, device=dev)            # the fused projection's rows
        q, k, v = x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:]
        wq, _ = rotated(q, qw, 1e-6, pos, fh, ah, True, ms)
        wk, _ = rotated(k, kw, 1e-6, pos, fh, ah, True, ms)
        wv = v.double().cpu().numpy()
        q_out, k_out = torch.empty(T, H, D, device=dev), torch.empty(T, Hkv, D, device=dev)
        pa.mrope_set_rows_kv(kp, vp, k, v, batch.slots, pos, fr, ax, q=q, q_out=q_out, k_out=k_out, q_norm=qw, k_norm=kw,
                             norm_eps=1e-6, mscale=ms, err_flag=err)
        prm = pa.PagedAttnParams(scale=scale)
        if step == 0:
            out = pa.prompt_attn(q_out, k_out, v, batch.query_start_loc, max(new), prm, row_end=row_end, err_flag=err)
        else:
            out = pa.build_paged_attn(q_out, kp, vp, Hkv, prm, batch)
        got, o = out.double().cpu().numpy(), 0
        for s in range(S):
            n = new[s]
            wp, we = walk(runs[s], computed[s] + n, True)
            assert np.array_equal(pos[:, o:o + n].cpu().numpy(), wp[:, computed[s]:])
            keys[s] = wk[o:o + n] if keys[s] is None else np.concatenate([keys[s], wk[o:o + n]])
            vals[s] = wv[o:o + n] if vals[s] is None else np.concatenate([vals[s], wv[o:o + n]])
            want = attend(wq[o:o + n], keys[s], vals[s], we[computed[s]:], scale)
            # the prompt in the rows' own precision; decodes within the paged kernels' tolerance over their pool
            tol = 3e-6 if step == 0 else 2e-3 if pool == F16 else 2e-5
            worst = (np.abs(got[o:o + n] - want).max(-1) / np.abs(want).max(-1)).max()
            assert worst <= tol, (step, s, worst)
            o += n
    assert int(err.item()) == 0
