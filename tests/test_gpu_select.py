"""Block selection and the attention over selected blocks on the GPU against
plain 64-bit implementations.

Tolerances count roundings.  Storing a result costs half a step of its type.  A
dot product of D float32 terms is off by at most (D + 8) 2^-24 times the sum of
its terms' magnitudes (also where the matrix cores add in another order); a
score's error e changes a weight by at most 2 e of it, a weight enters its
products with 22 bits or more, and a chain of n float32 additions adds n 2^-24.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

T = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-36, torch.bfloat16: 1e-36, torch.float16: 2.0 ** -24}
U = 2.0 ** -24
DEV = "cuda"


@pytest.fixture(scope="module")
def ext():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    import sparse_attention_cuda
    return sparse_attention_cuda


def rnd(seed, *shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)


def same(a, b):
    v = {2: torch.int16, 4: torch.int32}[a.element_size()]
    return torch.equal(a.view(v), b.view(v))


# ---------------------------------------------------------------- the lists

def select64(q, k, S, bs, causal, first, local):
    q, k = q.double().cpu(), k.double().cpu()
    B, N, H, D = q.shape
    Hkv = k.shape[2]
    nb = (N + bs - 1) // bs
    out = torch.full((B, N, Hkv, S), -1, dtype=torch.int32)
    j, own = torch.arange(nb)[None], (torch.arange(N) // bs)[:, None]
    ok = (j <= own) if causal else torch.ones(N, nb, dtype=torch.bool)
    forced = ok & ((j < first) | ((j <= own) & (j > own - local)))
    for b in range(B):
        for h in range(Hkv):
            mean = torch.stack([x.sum(0) / x.shape[0] for x in k[b, :, h].split(bs)])
            s = q[b].view(N, Hkv, H // Hkv, D)[:, h].sum(1) @ mean.t()
            s = torch.where(torch.isnan(s), torch.full_like(s, -math.inf), s)
            order = torch.sort(s, dim=-1, descending=True, stable=True).indices
            cls = torch.where(forced, 0, torch.where(ok, 1, 2))
            order = order.gather(1, torch.sort(cls.gather(1, order), dim=1, stable=True).indices)[:, :S]
            idx = torch.where(ok.gather(1, order), order, torch.full_like(order, nb)).sort(1).values
            out[b, :, h, :idx.shape[1]] = torch.where(idx < nb, idx, torch.full_like(idx, -1)).to(torch.int32)
    return out


SELECT = [
    # dtype, B, N, H, Hkv, D, bs, S, causal, first, local
    ("bf16", 1, 2048, 8, 8, 64, 64, 16, True, 1, 1),
    ("f32", 2, 1000, 4, 2, 64, 32, 8, True, 0, 1),
    ("f16", 1, 777, 6, 2, 128, 16, 12, False, 2, 3),
    ("bf16", 1, 5000, 3, 1, 40, 16, 64, True, 0, 2),   # 313 blocks: two chunks, the second carried into
    ("f32", 1, 9001, 1, 1, 16, 16, 5, False, 1, 4),    # 563 blocks: three chunks, 16 + 5 on one query
    ("f16", 3, 1, 2, 1, 8, 64, 3, True, 0, 1),
    ("f32", 1, 65, 2, 2, 24, 64, 1, True, 0, 1),
    ("bf16", 2, 130, 4, 4, 96, 64, 64, False, 0, 64),
]


@pytest.mark.parametrize("case", SELECT, ids=lambda c: "-".join(map(str, c)))
def test_select_blocks(ext, case):
    dt, B, N, H, Hkv, D, bs, S, causal, first, local = case
    q, k = rnd(1, B, N, H, D, dtype=T[dt]), rnd(2, B, N, Hkv, D, dtype=T[dt])
    got = ext.select_blocks(q, k, S, bs, causal, first, local)
    assert torch.equal(got.cpu(), select64(q, k, S, bs, causal, first, local))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_select_ties(ext, dt):
    """Zero queries, repeated blocks and scores that tie in float32 but not in
    float64; infinities and NaN."""
    N, bs, D = 6000, 16, 64  # 375 blocks: ties within a chunk and across two
    q, k = rnd(1, 1, N, 2, D, dtype=T[dt]), rnd(2, 1, N, 1, D, dtype=T[dt])
    q[:, ::5] = 0
    k[:, :3000] = k[:, :16].repeat(1, 188, 1, 1)[:, :3000]  # equal blocks
    for causal in (True, False):
        assert torch.equal(ext.select_blocks(q, k, 9, bs, causal).cpu(), select64(q, k, 9, bs, causal, 0, 1))
    k[0, 50, 0, 3], k[0, 3100, 0, 5], k[0, 5000, 0, 7] = math.inf, -math.inf, math.nan
    q[0, 4000, 1, 5], q[0, 4001, 0, 0] = math.inf, math.nan
    for causal in (True, False):
        assert torch.equal(ext.select_blocks(q, k, 9, bs, causal).cpu(), select64(q, k, 9, bs, causal, 0, 1))


def test_select_near_ties(ext):
    """Blocks whose scores differ by less than a float32 step."""
    N, bs, D, nb = 640, 16, 16, 40
    q, k = torch.zeros(1, N, 1, D, device=DEV), torch.zeros(1, N, 1, D, device=DEV)
    q[..., 0], q[..., 1] = 1.0, 1.0
    k[..., 0] = 1024.0
    tiny = torch.tensor([(7 * i) % nb for i in range(nb)], dtype=torch.float32, device=DEV) * 2.0 ** -30
    k[..., 1] = tiny.repeat_interleave(bs)[None, :, None]
    for S in (1, 4, 13):
        assert torch.equal(ext.select_blocks(q, k, S, bs, False).cpu(), select64(q, k, S, bs, False, 0, 1))


# ---------------------------------------------------------------- attention

def mask_of(blocks, H, bs, causal):
    """[B, H, N, N] of the listed keys."""
    B, N, Hkv, S = blocks.shape
    nb = (N + bs - 1) // bs
    t = blocks.long().cpu()
    t = torch.where((t < 0) | (t >= nb), torch.full_like(t, nb), t)
    hit = torch.zeros(B, N, Hkv, nb + 1, dtype=torch.bool).scatter_(-1, t, True)
    m = hit[..., torch.arange(N) // bs].permute(0, 2, 1, 3).repeat_interleave(H // Hkv, 1)
    return m & torch.ones(N, N, dtype=torch.bool).tril() if causal else m


def attend64(q, k, v, g, blocks, bs, causal, scale=None, dtype=None, stored_o=True):
    """o, lse, dq, dk, dv in float64 and bounds of the errors of o, dq, dk, dv."""
    half, tiny = HALF[q.dtype], TINY[q.dtype]
    qd, kd, vd, gd = (x.double().cpu().transpose(1, 2) for x in (q, k, v, g))
    B, H, N, D = qd.shape
    G = H // kd.shape[1]
    sc = scale or D ** -0.5
    kd, vd = kd.repeat_interleave(G, 1), vd.repeat_interleave(G, 1)
    m = mask_of(blocks, H, bs, causal)
    s = (qd @ kd.transpose(-1, -2)) * sc
    live = m.any(-1, keepdim=True)
    sm = s.masked_fill(~m, -math.inf)
    p = torch.where(live, torch.softmax(sm, -1), torch.zeros_like(s))
    p = torch.nan_to_num(p)
    o = p @ vd
    lse = torch.logsumexp(sm, -1) / math.log(2)
    dp = gd @ vd.transpose(-1, -2)
    delta = (gd * o).sum(-1, keepdim=True)
    ds = p * (dp - delta) * sc
    dq, dk, dv = ds @ kd, ds.transpose(-1, -2) @ qd, p.transpose(-1, -2) @ gd
    # errors
    a = lambda x: x.abs()  # noqa: E731
    e_s = ((D + 8) * U * (a(qd) @ a(kd).transpose(-1, -2)) * sc).masked_fill(~m, 0).amax(-1, keepdim=True) + 2.0 ** -21
    keys = m.sum(-1, keepdim=True).double()
    rel_p = 2 * e_s + 2.0 ** -21 + (keys / 16 + 64) * U + 2.0 ** -23 * a(lse)[..., None].nan_to_num(0, 0, 0)
    b_o = half * a(o) + rel_p * (p @ a(vd)) + tiny
    e_dp = (D + 8) * U * (a(gd) @ a(vd).transpose(-1, -2))
    e_dl = (gd.abs() * (half * a(o) + rel_p * (p @ a(vd)))).sum(-1, keepdim=True) + (D + 8) * U * (a(gd) * a(o)).sum(-1, keepdim=True)
    e_ds = p * (rel_p * a(dp - delta) + e_dp + e_dl) * sc + 2.0 ** -21 * a(ds)
    rows = m.sum(-2).double()[..., None]
    b_dq = half * a(dq) + e_ds @ a(kd) + (keys / 16 + 64) * U * (a(ds) @ a(kd)) + tiny
    t = lambda x: x.transpose(-1, -2)  # noqa: E731
    chain = (rows * G + 64) * U
    e_dk = t(e_ds) @ a(qd) + chain * (t(a(ds)) @ a(qd))
    e_dv = t(rel_p * p) @ a(gd) + chain * (t(p) @ a(gd))
    grp = lambda x: x.view(B, -1, G, N, D).sum(2)  # noqa: E731
    dk, dv, e_dk, e_dv = (grp(x) for x in (dk, dv, e_dk, e_dv))
    back = lambda x: x.transpose(1, 2)  # noqa: E731
    return dict(o=(back(o), back(b_o)), dq=(back(dq), back(b_dq)), dk=(back(dk), back(half * a(dk) + e_dk + tiny)),
                dv=(back(dv), back(half * a(dv) + e_dv + tiny)), lse=lse.transpose(1, 2))


def close(name, got, ref):
    val, bound = ref
    got = got.double().cpu()
    assert bool(torch.isfinite(got).all()), name
    worst = float(((got - val).abs() / bound).max()) if got.numel() else 0.0
    print(f"  {name}: worst error / bound {worst:.3f}", flush=True)
    assert worst <= 1.0, (name, worst)


def wild_table(seed, B, N, Hkv, S, nb):
    """Unordered lists with repeats, padding anywhere, blocks outside, blocks behind
    the query, empty lists; block 0 in most of them."""
    g = torch.Generator().manual_seed(seed)
    t = torch.randint(-2, nb + 2, (B, N, Hkv, S), generator=g, dtype=torch.int32)
    t[..., 0] = torch.where(torch.rand((B, N, Hkv), generator=g) < 0.7, torch.zeros_like(t[..., 0]), t[..., 0])
    t[torch.rand((B, N, Hkv), generator=g) < 0.05] = -1
    t[:, N // 2, :, :] = 1 << 30
    return t.to(DEV)


ATTEND = [
    # dtype, B, N, H, Hkv, D, bs, S, causal
    ("f32", 1, 300, 2, 2, 64, 64, 4, True),
    ("bf16", 2, 333, 4, 2, 64, 64, 3, True),
    ("f16", 1, 500, 6, 2, 64, 32, 5, False),
    ("bf16", 1, 400, 5, 1, 128, 64, 4, True),     # five heads on one: tiles that end inside a pair's heads
    ("f16", 1, 257, 3, 3, 128, 16, 8, True),
    ("f32", 2, 190, 4, 1, 128, 32, 3, False),
    ("bf16", 1, 700, 1, 1, 32, 16, 6, True),
    ("f32", 1, 321, 2, 1, 8, 64, 2, True),
    ("f16", 1, 129, 2, 2, 80, 64, 64, False),
    ("bf16", 3, 65, 2, 2, 48, 32, 1, True),
    ("f32", 1, 1, 1, 1, 16, 16, 1, True),
    ("f16", 2, 15, 8, 4, 24, 64, 2, False),
    ("f32", 1, 200, 32, 1, 40, 16, 4, True),
    ("f16", 1, 1500, 2, 1, 64, 64, 16, True),
]


@pytest.mark.parametrize("case", ATTEND, ids=lambda c: "-".join(map(str, c)))
def test_forward_and_gradients(ext, case):
    dt, B, N, H, Hkv, D, bs, S, causal = case
    dtype, nb = T[dt], (N + bs - 1) // bs
    q, g = rnd(1, B, N, H, D, dtype=dtype), rnd(4, B, N, H, D, dtype=dtype)
    k, v = rnd(2, B, N, Hkv, D, dtype=dtype), rnd(3, B, N, Hkv, D, dtype=dtype)
    blocks = wild_table(5, B, N, Hkv, S, nb)
    ref = attend64(q, k, v, g, blocks, bs, causal)
    out, lse = ext.selected_forward(q, k, v, blocks, bs, causal, return_lse=True)
    close("out", out, ref["o"])
    dead = ref["lse"] == -math.inf
    lc = lse.double().cpu()
    assert bool((lc[dead] == -math.inf).all()) and not bool(out.cpu()[dead].any())
    assert bool(((lc - ref["lse"]).abs()[~dead] <= 1e-5 * (1 + ref["lse"].abs()[~dead])).all())
    assert same(out, ext.selected_forward(q, k, v, blocks, bs, causal))
    grads = ext.selected_backward(q, k, v, g, blocks, bs, causal, out=out, lse=lse)
    for n, x in zip(("dq", "dk", "dv"), grads):
        close(n, x, ref[n])
    for x, y in zip(grads, ext.selected_backward(q, k, v, g, blocks, bs, causal)):
        assert same(x, y)  # from its own forward, and the same bits every time


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_scale_small_gradients_and_peaked_rows(ext, dt):
    dtype, B, N, H, bs = T[dt], 1, 256, 2, 64
    q, k, v, g = (rnd(i, B, N, H, 64, dtype=dtype) for i in range(1, 5))
    q = (q.float() * 8).to(dtype)
    g[:, ::2] *= 1e-3
    g[:, 1::16] *= 100
    blocks = wild_table(5, B, N, H, 4, 4)
    for scale in (None, 0.02):
        ref = attend64(q, k, v, g, blocks, bs, True, scale)
        out, lse = ext.selected_forward(q, k, v, blocks, bs, True, True, scale)
        close("out", out, ref["o"])
        for n, x in zip(("dq", "dk", "dv"), ext.selected_backward(q, k, v, g, blocks, bs, True, out, lse, scale)):
            close(n, x, ref[n])


def test_gradients_against_differences(ext):
    """Directional derivatives of the 64-bit loss by central differences."""
    B, N, H, Hkv, D, bs = 1, 150, 4, 2, 32, 32
    x = [rnd(i, B, N, h, D) for i, h in ((1, H), (2, Hkv), (3, Hkv))]
    g = rnd(4, B, N, H, D)
    blocks = wild_table(5, B, N, Hkv, 3, 5)
    grads = ext.selected_backward(*x, g, blocks, bs, True)
    for i in range(3):
        d = rnd(10 + i, *x[i].shape)
        vals = []
        for sgn in (1, -1):
            y = [t.double() for t in x]
            y[i] = y[i] + sgn * 1e-5 * d.double()
            m = mask_of(blocks, H, bs, True)
            qd, kd, vd = (t.cpu().transpose(1, 2) for t in y)
            kd, vd = kd.repeat_interleave(2, 1), vd.repeat_interleave(2, 1)
            s = (qd @ kd.transpose(-1, -2) * D ** -0.5).masked_fill(~m, -math.inf)
            p = torch.nan_to_num(torch.softmax(s, -1))
            vals.append(float(((p @ vd) * g.double().cpu().transpose(1, 2)).sum()))
        diff = (vals[0] - vals[1]) / 2e-5
        mine = float((grads[i].double() * d.double()).sum())
        scale = float((grads[i].double().abs() * d.double().abs()).sum())
        assert abs(mine - diff) <= 1e-5 * scale, (i, mine, diff)


@pytest.mark.parametrize("dt,bs,D", [("f32", 64, 64), ("bf16", 32, 64), ("f16", 16, 32), ("bf16", 64, 128)])
def test_values_behind_a_query_do_not_reach_it(ext, dt, bs, D):
    """Infinite and NaN keys, values, queries and gradients: every row and key that
    does not attend them is as without them."""
    dtype, B, N, H = T[dt], 1, 3 * bs - 5, 2
    nb = 3
    q, k, v, g = (rnd(i, B, N, H, D, dtype=dtype) for i in range(1, 5))
    blocks = torch.arange(nb, dtype=torch.int32, device=DEV).expand(B, N, H, nb).contiguous()
    at = bs + bs // 2  # inside the second block
    clean_o, clean_l = ext.selected_forward(q, k, v, blocks, bs, True, True)
    for who in "kvqg":
        for val in (math.nan, math.inf, -math.inf):
            x = dict(q=q.clone(), k=k.clone(), v=v.clone(), g=g.clone())
            x[who][0, at, 0, 3] = val
            o, lse = ext.selected_forward(x["q"], x["k"], x["v"], blocks, bs, True, True)
            o2 = o.clone()
            o2[:, at:, 0] = clean_o[:, at:, 0]
            close("out", o2, (clean_o.double().cpu(), 2 * HALF[dtype] * clean_o.double().cpu().abs() + 1e-5))
            grads = ext.selected_backward(x["q"], x["k"], x["v"], x["g"], blocks, bs, True, out=o, lse=lse)
            # without the bad rows' and keys' pairs: queries before `at` see none of it; the other head neither
            ref = attend64(q, k, v, g, blocks, bs, True)
            dq = grads[0].clone()
            dq[:, at:, 0] = ref["dq"][0][:, at:, 0].to(dtype).to(DEV)
            close("dq", dq, ref["dq"])
            if who in "qg":  # one row: keys behind it get nothing of it
                assert bool(torch.isfinite(grads[0][:, at + 1:]).all())
                for n, y in zip(("dk", "dv"), grads[1:]):
                    y = y.clone()
                    y[:, :at + 1, 0] = ref[n][0][:, :at + 1, 0].to(dtype).to(DEV)
                    close(n, y, ref[n])
            else:  # rows from `at` on are spoilt, and with them what they add to every key they see
                for n, y in zip(("dk", "dv"), grads[1:]):
                    assert bool(torch.isfinite(y[:, :, 1]).all())


def test_rows_of_infinite_scores(ext):
    """-inf scores take no weight; a row of nothing else, and +inf, are undefined."""
    N, bs = 96, 32
    q, k, v = (rnd(i, 1, N, 1, 32) for i in range(1, 4))
    q[:] = 0
    q[..., 0] = 1
    k[:, 10, :, 0] = -math.inf
    blocks = torch.arange(3, dtype=torch.int32, device=DEV).expand(1, N, 1, 3).contiguous()
    out = ext.selected_forward(q, k, v, blocks, bs, False)
    s = (q[0, :, 0].double() @ k[0, :, 0].nan_to_num(0, 0, 0).double().t())
    s[:, 10] = -math.inf
    s = s * 32 ** -0.5
    ref = torch.softmax(s, -1) @ v[0, :, 0].double()
    assert float((out[0, :, 0].double() - ref).abs().max()) < 1e-5
    k[..., 0] = -math.inf
    assert bool(torch.isnan(ext.selected_forward(q, k, v, blocks, bs, False)).all())
    k[..., 0] = 0
    k[:, 40, :, 0] = math.inf
    out = ext.selected_forward(q, k, v, blocks, bs, True)
    assert bool(torch.isnan(out[:, 40:]).all()) and bool(torch.isfinite(out[:, :40]).all())


def test_many_heads_run_in_groups(ext, monkeypatch):
    """More partial rows than are kept at once: groups of heads one after another,
    the same results as head by head."""
    B, N, H, D, bs, S = 1, 8192, 24, 128, 64, 16  # 24 x 67 MB of partial rows
    q, k, v, g = (rnd(i, B, N, H, D, dtype=torch.bfloat16) for i in range(1, 5))
    blocks = ext.select_blocks(q, k, S, bs)
    out, lse = ext.selected_forward(q, k, v, blocks, bs, True, True)
    grads = ext.selected_backward(q, k, v, g, blocks, bs, True, out, lse)
    for h in (0, 15, 23):
        one = [x[:, :, h:h + 1].contiguous() for x in (q, k, v, blocks, g)]
        o1, l1 = ext.selected_forward(*one[:4], bs, True, True)
        assert float((o1 - out[:, :, h:h + 1]).abs().max()) <= 2.0 ** -7
        for x, y in zip(ext.selected_backward(*one[:3], one[4], one[3], bs, True, o1, l1), grads):
            y = y[:, :, h:h + 1]
            assert bool(((x - y).abs() <= 2.0 ** -7 * y.abs() + 2e-3).all())


def test_all_blocks_is_dense_attention(ext):
    N, H, D = 512, 4, 64
    q, k, v, g = (rnd(i, 1, N, H, D) for i in range(1, 5))
    blocks = ext.select_blocks(q, k, 8)
    assert torch.equal(blocks[0, :, 0].cpu(), torch.tensor(
        [[j if j <= i // 64 else -1 for j in range(8)] for i in range(N)], dtype=torch.int32))
    out = ext.selected_forward(q, k, v, blocks)
    assert float((out - ext.dense_forward(q, k, v, True)).abs().max()) < 1e-5
    for a, b in zip(ext.selected_backward(q, k, v, g, blocks), ext.dense_backward(q, k, v, g, True)):
        assert float((a - b).abs().max()) < 1e-4


# ---------------------------------------------------------------- together

@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_layer_trains_and_infers(ext, dt):
    """MACoreAttention(pattern="block_select") against its PyTorch path."""
    from layers.ma_core_bridge import MACoreAttention
    dtype = T[dt]
    kw = dict(pattern="block_select", num_selected=4, block_size=32, causal=True, first_blocks=1)
    layer = MACoreAttention(fallback_training=False, **kw).train()
    x = [rnd(i, 2, 300, 4, 64, dtype=dtype).requires_grad_(True) for i in range(1, 4)]
    g = rnd(4, 2, 300, 4, 64, dtype=dtype)
    out = layer(*x)
    out.backward(g)
    plain = MACoreAttention(**kw).train()  # fallback_training: the PyTorch path
    y = [t.detach().clone().requires_grad_(True) for t in x]
    ref = plain(*y)
    ref.backward(g)
    tol = 1e-4 if dt == "f32" else 3e-2
    assert float((out - ref).detach().float().abs().max()) <= tol
    for a, b in zip(x, y):
        assert bool(((a.grad - b.grad).float().abs() <= tol * (1 + b.grad.float().abs())).all())
    with torch.no_grad():
        assert same(layer.eval()(*x), out.detach())
    # gradients of some inputs only
    z = [t.detach().clone() for t in x]
    z[1].requires_grad_(True)
    layer.train()(*z).backward(g)
    assert same(z[1].grad, x[1].grad) and z[0].grad is None


def test_prompt_then_tokens_equal_the_whole_sequence(ext):
    """The prompt on select_blocks / selected_forward, single tokens on the paged
    cache's forms: every row as the whole sequence at once gives it."""
    import paged_attention as pa
    B, N, P, H, Hkv, D, bs, S, dtype = 2, 330, 300, 4, 2, 64, 32, 4, torch.float32
    q, k, v = (rnd(i, B, N, h, D, dtype=dtype) for i, h in ((1, H), (2, Hkv), (3, Hkv)))
    blocks = ext.select_blocks(q, k, S, bs, True, first_blocks=1)
    whole = ext.selected_forward(q, k, v, blocks, bs, True)
    cache = pa.PagedCache(B * 11 + 1, bs, Hkv, D, dtype, DEV, key_sums=True)
    table = torch.randperm(B * 11, generator=torch.Generator().manual_seed(1)).view(B, 11).to(torch.int32).to(DEV)
    at = torch.zeros(B, dtype=torch.int32, device=DEV)
    pa.paged_append(cache, k[:, :P].contiguous(), v[:, :P].contiguous(), table, at)
    at += P
    for i in range(P, N):
        row = slice(i, i + 1)
        pa.paged_append(cache, k[:, row].contiguous(), v[:, row].contiguous(), table, at)
        at += 1
        pages = pa.paged_select(q[:, i].contiguous(), cache, table, at, S, first_pages=1)
        assert torch.equal(pages, blocks[:, i])
        got = pa.paged_decode(q[:, i].contiguous(), cache, table, at, pages=pages)
        assert float((got - whole[:, i]).abs().max()) < 1e-5


def test_graph_replays(ext):
    """A training step's calls in a graph: replays with new inputs equal the eager
    calls, with eager work and synchronisations in between; two graphs in turn."""
    B, N, H, D, bs, S, dtype = 1, 700, 4, 64, 64, 5, torch.float16
    bufs = [rnd(i, B, N, H, D, dtype=dtype) for i in range(1, 5)]

    def step(q, k, v, g):
        blocks = ext.select_blocks(q, k, S, bs)
        out, lse = ext.selected_forward(q, k, v, blocks, bs, True, True)
        return [blocks, out, *ext.selected_backward(q, k, v, g, blocks, bs, True, out, lse)]

    step(*bufs)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step(*bufs)
        graphs.append((gr, out))
    for r in range(6):
        for i in range(4):
            bufs[i].copy_(rnd(50 + 4 * r + i, B, N, H, D, dtype=dtype))
        gr, out = graphs[r % 2]
        gr.replay()
        ref = step(*bufs)
        torch.cuda.synchronize()
        assert torch.equal(out[0], ref[0])
        for a, b in zip(out[1:], ref[1:]):
            assert same(a, b), r


def test_other_stream_and_events(ext):
    q, k, v = (rnd(i, 1, 900, 2, 64, dtype=torch.bfloat16) for i in range(1, 4))
    blocks = ext.select_blocks(q, k, 4)
    ref = ext.selected_forward(q, k, v, blocks)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b2 = ext.select_blocks(q, k, 4)
        got = ext.selected_forward(q, k, v, b2)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(b2, blocks) and same(got, ref)
    e = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
    for x in e:
        x.record()
    torch.cuda.synchronize()
    for call in (lambda: ext.select_blocks(q, k, 4), lambda: ext.selected_forward(q, k, v, blocks),
                 lambda: ext.selected_backward(q, k, v, q, blocks, out=ref, lse=torch.zeros(1, 900, 2, device=DEV))):
        with ext.kernel_events(*e):
            call()
        torch.cuda.synchronize()
        assert 0.0 < e[0].elapsed_time(e[1]) < 100.0


def test_refusals(ext):
    q = rnd(1, 1, 100, 4, 64, dtype=torch.bfloat16)
    k = rnd(2, 1, 100, 2, 64, dtype=torch.bfloat16)
    b = torch.zeros(1, 100, 2, 3, dtype=torch.int32, device=DEV)
    bad = [
        (lambda: ext.select_blocks(q, k.float(), 3), "dtype"),
        (lambda: ext.select_blocks(q, k[:, :99].contiguous(), 3), "sequence length"),
        (lambda: ext.select_blocks(q[:, :, :3].contiguous(), k, 3), "multiple"),
        (lambda: ext.select_blocks(q.transpose(1, 2), k, 3), "contiguous"),
        (lambda: ext.select_blocks(q, k, 0), "num_selected"),
        (lambda: ext.select_blocks(q, k, 3, first_blocks=3), "fit"),
        (lambda: ext.select_blocks(q, k, 3, block_size=128), "block_size"),
        (lambda: ext.selected_forward(q, k, k[:, :, :1].contiguous(), b), "same shape"),
        (lambda: ext.selected_forward(q, k, k, b.long()), "int32"),
        (lambda: ext.selected_forward(q, k, k, b[..., :1, :].contiguous()), "blocks must be"),
        (lambda: ext.selected_forward(q, k, k, b.cpu()), "blocks must be"),
        (lambda: ext.selected_forward(q, k, k, b, scale=-1.0), "scale"),
        (lambda: ext.selected_backward(q, k, k, k, b), "same shape"),
        (lambda: ext.selected_backward(q, k, k, q, b, out=q, lse=q[..., 0].contiguous()), "lse"),
        (lambda: ext.selected_forward(*(rnd(1, 1, 100, 2, 60, dtype=torch.bfloat16),) * 3, b), "head_dim"),
    ]
    import re
    for call, msg in bad:
        with pytest.raises(RuntimeError) as e:
            call()
        assert re.search(msg, str(e.value)), (msg, str(e.value))
    # empty batches and sequences
    for shape in ((0, 100, 2, 64), (1, 0, 2, 64)):
        x = torch.zeros(shape, device=DEV)
        bl = ext.select_blocks(x, x, 3)
        assert bl.shape == (*shape[:2], 2, 3)
        assert ext.selected_forward(x, x, x, bl).shape == shape
        assert all(t.shape == shape for t in ext.selected_backward(x, x, x, x, bl))


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_padded_batch(ext, dt):
    """Sequences padded behind their ends: the rows before are those of the
    unpadded sequence (causal: nothing behind a row reaches it), bit by bit with
    zeros behind them.  With NaN the rows of the block that holds the end are
    summed key by key, in another order: they are held to the 64-bit result."""
    B, N, n, H, D, bs, S = 2, 500, 333, 2, 64, 32, 4
    q, k, v, g = (rnd(i, B, N, H, D, dtype=T[dt]) for i in range(1, 5))
    short = [x[:, :n].contiguous() for x in (q, k, v, g)]
    bl = ext.select_blocks(short[0], short[1], S, bs)
    o, lse = ext.selected_forward(*short[:3], bl, bs, True, True)
    grads = ext.selected_backward(*short[:3], short[3], bl, bs, True, o, lse)
    for fill in (0.0, math.nan):
        x = [t.clone() for t in (q, k, v, g)]
        for t in x:
            t[:, n:] = fill
        if fill == 0.0:  # rows whose every score ties
            full = ext.select_blocks(x[0], x[1], S, bs)
            assert torch.equal(full.cpu(), select64(x[0], x[1], S, bs, True, 0, 1))
        pad = torch.full((B, N, H, S), -1, dtype=torch.int32, device=DEV)
        pad[:, :n] = bl
        po, pl = ext.selected_forward(x[0], x[1], x[2], pad, bs, True, True)
        pg = ext.selected_backward(x[0], x[1], x[2], x[3], pad, bs, True, po, pl)
        ref = attend64(*short, bl, bs, True)
        for name, a, b in zip(("o", "dq", "dk", "dv"), (po, *pg), (o, *grads)):
            assert not bool(a[:, n:].any()), name
            close(name, a[:, :n], ref[name])
            if fill == 0.0:
                assert same(a[:, :n].contiguous(), b), name


def test_two_streams_at_once(ext):
    """Two training steps in flight on two streams do not meet."""
    sets = [[rnd(10 * j + i, 1, 3000, 4, 64, dtype=torch.float16) for i in range(4)] for j in range(2)]

    def step(q, k, v, g):
        bl = ext.select_blocks(q, k, 8)
        o, l = ext.selected_forward(q, k, v, bl, return_lse=True)
        return [o, *ext.selected_backward(q, k, v, g, bl, out=o, lse=l)]

    ref = [step(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = []
        for s, st in zip(sets, streams):
            with torch.cuda.stream(st):
                got.append(step(*s))
        torch.cuda.synchronize()
        for a, b in zip(got, ref):
            assert all(same(x, y) for x, y in zip(a, b))
