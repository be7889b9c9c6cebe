"""Paged cache on the GPU against plain 64-bit implementations.

Tolerances count roundings: storing a result costs half a step of its type;
a score's float32 error e is at most (head_dim + 8) 2^-24 sum |q_d k_d| scale,
which changes a weight by at most 2 e of it (its own and the denominator's),
and a chain of float32 additions adds 2^-24 per link.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

T = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -24}
DEV = "cuda"


@pytest.fixture(scope="module")
def pa():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    import paged_attention
    return paged_attention


def rnd(seed, *shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)


def tables(seed, B, width, pages):
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(pages, generator=g)[:B * width].view(B, width).to(torch.int32).to(DEV)


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# ---------------------------------------------------------------- append

def rotate64(x, pos, freq, interleaved):
    """x [B, N, h, D] -> float64, on the host."""
    x = x.double().cpu().clone()
    R = 2 * freq.numel()
    a = pos.double().cpu()[:, :, None, None] * freq.cpu()
    if interleaved:
        x0, x1 = x[..., 0:R:2].clone(), x[..., 1:R:2].clone()
        x[..., 0:R:2], x[..., 1:R:2] = x0 * a.cos() - x1 * a.sin(), x0 * a.sin() + x1 * a.cos()
    else:
        x0, x1 = x[..., :R // 2].clone(), x[..., R // 2:R].clone()
        x[..., :R // 2], x[..., R // 2:R] = x0 * a.cos() - x1 * a.sin(), x0 * a.sin() + x1 * a.cos()
    return x


def same(a, b):
    """Bit equality, NaN included."""
    v = {2: torch.int16, 4: torch.int32, 8: torch.int64}[a.element_size()]
    return torch.equal(a.view(v), b.view(v))


APPEND = [
    # dtype, D, rotated, interleaved, Hkv, H, page, N, starts, counts, sums
    ("bf16", 64, 64, False, 4, 8, 64, 1, [0, 63, 64, 500], None, True),
    ("f16", 64, 32, False, 3, 3, 16, 37, [0, 5, 15, 16], [37, 0, 1, 36], True),
    ("f32", 128, 128, True, 2, 8, 32, 70, [31, 0], [70, 69], True),
    ("f32", 8, 0, False, 1, 1, 16, 3, [14], None, True),
    ("bf16", 80, 80, False, 5, 10, 48, 65, [47, 100000], [64, 65], False),
    ("f16", 40, 16, True, 1, 4, 128, 130, [1], None, True),
    ("bf16", 128, 64, False, 1, 12, 16, 17, [3, 9], None, False),
    ("f32", 24, 16, False, 2, 2, 64, 129, [0, 1 << 20], [129, 3], True),
    ("bf16", 64, 64, False, 2, 4, 1024, 1500, [1000, 0], [1500, 24], True),  # pages longer than a tile of tokens
    ("f16", 128, 128, False, 40, 80, 16, 18, [5], None, True),               # a token of more units than threads
]


@pytest.mark.parametrize("case", APPEND, ids=lambda c: f"{c[0]}-D{c[1]}-R{c[2]}-p{c[6]}-N{c[7]}")
def test_append(pa, case):
    dt, D, R, inter, Hkv, H, page, N, starts, counts, sums = case
    dtype, B = T[dt], len(starts)
    # far positions live in a short table: logical pages are taken modulo nothing, so the table is wide
    width = (max(starts) + N + page - 1) // page
    far = width > 64
    pages = B * min(width, 64) + 2
    if far:  # only the pages that the call touches point into the cache
        table = torch.full((B, width), -1, dtype=torch.int32)
        nxt = iter(torch.randperm(pages, generator=torch.Generator().manual_seed(1)).tolist())
        for b, s in enumerate(starts):
            for l in range(s // page, (s + N - 1) // page + 1):
                table[b, l] = next(nxt)
        table = table.to(DEV)
    else:
        table = tables(1, B, width, pages)
    k0, v0 = rnd(2, pages, page, Hkv, D, dtype=dtype), rnd(3, pages, page, Hkv, D, dtype=dtype)
    s0 = rnd(4, pages, Hkv, D)
    cache = pa.PagedCache.from_tensors(k0.clone(), v0.clone(), s0.clone() if sums else None)
    k, v, q = rnd(5, B, N, Hkv, D, dtype=dtype), rnd(6, B, N, Hkv, D, dtype=dtype), rnd(7, B, N, H, D, dtype=dtype)
    n = counts or [N] * B
    for b in range(B):  # rows behind a stream's count are padding: nothing of them may be stored
        k[b, n[b]:], v[b, n[b]:] = float("nan"), float("nan")
    start = i32(*starts)
    rot = pa.Rotation(R, interleaved=inter, device=DEV) if R else None
    out = pa.paged_append(cache, k, v, table, start, counts=i32(*counts) if counts else None, rotation=rot, query=q)
    pos = start[:, None].long() + torch.arange(N, device=DEV)
    freq = rot.inv_freq if R else torch.zeros(0, dtype=torch.float64)
    eps = HALF[dtype] * (1 + 2.0 ** -10)  # a result passes through float32 on its way to 16 bits

    def close(name, got, ref):
        err = (got.double().cpu() - ref).abs()
        worst = float((err / (eps * ref.abs() + TINY[dtype] + 1e-15)).max())
        print(f"  {name}: worst error / bound {worst:.3f}", flush=True)
        assert worst <= 1.0

    close("query", out, rotate64(q, pos, freq, inter))
    kr = rotate64(k, pos, freq, inter)
    wk, wv = k0.clone(), v0.clone()
    got_k, got_v = cache.key.cpu(), cache.value.cpu()
    stored = torch.zeros(pages, page, dtype=torch.bool)
    touched = {}
    t = table.cpu()
    for b in range(B):
        for i in range(n[b]):
            p, s = int(t[b, (starts[b] + i) // page]), (starts[b] + i) % page
            stored[p, s] = True
            touched[p] = max(touched.get(p, 0), s + 1)
            wv[p, s] = v[b, i]
            kr_row = kr[b, i]
            err = (got_k[p, s].double() - kr_row).abs()
            assert bool((err <= eps * kr_row.abs() + TINY[dtype] + 1e-15).all()), (b, i)
    assert same(got_v, wv.cpu())
    assert same(got_k[~stored], wk.cpu()[~stored])
    if sums:
        got_s = cache.key_sums.cpu()
        for p in range(pages):
            if p not in touched:
                assert same(got_s[p], s0[p].cpu()), p
                continue
            x = got_k[p, :touched[p]].double()
            bound = touched[p] * 2.0 ** -24 * x.abs().sum(0) + 1e-30
            assert bool(((got_s[p].double() - x.sum(0)).abs() <= bound).all()), p


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_append_token_by_token_equals_at_once(pa, dt):
    """Bitwise, page sums too; and a stream set back and appended to again."""
    dtype, B, N, Hkv, D, page = T[dt], 2, 41, 2, 64, 16
    k, v = rnd(1, B, N, Hkv, D, dtype=dtype), rnd(2, B, N, Hkv, D, dtype=dtype)
    table = tables(3, B, 4, 9)
    rot = pa.Rotation(64, device=DEV)
    base = rnd(4, 9, page, Hkv, D, dtype=dtype), rnd(5, 9, page, Hkv, D, dtype=dtype), rnd(6, 9, Hkv, D)
    caches = [pa.PagedCache.from_tensors(*(x.clone() for x in base)) for _ in range(3)]
    starts = torch.tensor([7, 0])
    pa.paged_append(caches[0], k, v, table, starts.int().to(DEV), rotation=rot)
    for i in range(N):
        pa.paged_append(caches[1], k[:, i:i + 1].contiguous(), v[:, i:i + 1].contiguous(), table,
                        (starts + i).int().to(DEV), rotation=rot)
    other = rnd(9, B, N, Hkv, D, dtype=dtype)
    pa.paged_append(caches[2], other, other, table, starts.int().to(DEV), rotation=rot)
    pa.paged_append(caches[2], k[:, :30].contiguous(), v[:, :30].contiguous(), table, starts.int().to(DEV), rotation=rot)
    pa.paged_append(caches[2], k[:, 30:].contiguous(), v[:, 30:].contiguous(), table, (starts + 30).int().to(DEV),
                    rotation=rot)
    for c in caches[1:]:
        assert same(c.key, caches[0].key) and same(c.value, caches[0].value) and same(c.key_sums, caches[0].key_sums)


def test_append_skips_what_the_tables_do_not_hold(pa):
    """Pages outside the cache, positions behind the table, negative counts."""
    B, N, Hkv, D, page = 4, 20, 1, 16, 16
    k = rnd(1, B, N, Hkv, D)
    table = i32(0, 99, -5, 1, 2, 3, 4, 5).view(4, 2)
    cache = pa.PagedCache.from_tensors(torch.zeros(6, page, Hkv, D, device=DEV), torch.zeros(6, page, Hkv, D, device=DEV),
                                       torch.full((6, Hkv, D), -1.0, device=DEV))
    pa.paged_append(cache, k, k, table, i32(0, 0, 30, -7), counts=i32(20, 20, 20, -1))
    got = cache.key.cpu()
    kc = k.cpu()
    assert torch.equal(got[0], kc[0, :16]) and torch.equal(got[1, :4], kc[1, 16:]) and not got[1, 4:].any()
    assert torch.equal(got[3, 14:], kc[2, :2]) and not got[2].any()  # stream 2 starts in its second page
    assert not got[4].any() and not got[5].any()
    s = cache.key_sums.cpu()
    assert (s[2] == -1).all() and (s[4:] == -1).all() and not (s[0] == -1).any() and not (s[3] == -1).any()


# ---------------------------------------------------------------- decode

def key_sets(lengths, Hkv, page, left, nglobal, pages):
    """[B][Hkv] ascending token lists."""
    out = []
    for b, n in enumerate(lengths):
        rows = []
        for h in range(Hkv):
            if pages is not None:
                keep = sorted({int(p) for p in pages[b, h] if 0 <= int(p) and int(p) * page < n})
                rows.append([t for p in keep for t in range(p * page, min(n, (p + 1) * page))])
            elif left is not None:
                rows.append([t for t in range(n) if t >= n - 1 - left or t < nglobal])
            else:
                rows.append(list(range(n)))
        out.append(rows)
    return out


def decode64(q, cache, table, sets, scale=None):
    """(out, bound, lse) in float64 on the host."""
    q, ck, cv, t = q.double().cpu(), cache.key.cpu(), cache.value.cpu(), table.cpu()
    B, H, D = q.shape
    page, Hkv = ck.shape[1], ck.shape[2]
    G = H // Hkv
    scale = scale or D ** -0.5
    out, bound = torch.zeros(B, H, D, dtype=torch.float64), torch.zeros(B, H, D, dtype=torch.float64)
    lse = torch.full((B, H), -math.inf, dtype=torch.float64)
    lse_bound = torch.zeros(B, H, dtype=torch.float64)
    half = HALF[cache.key.dtype]
    for b in range(B):
        for h in range(H):
            toks = [x for x in sets[b][h // G] if 0 <= int(t[b, x // page]) < ck.shape[0]]
            if not toks:
                continue
            tok = torch.tensor(toks)
            phys = t[b, tok // page].long()
            k, v = ck[phys, tok % page, h // G].double(), cv[phys, tok % page, h // G].double()
            s = k @ q[b, h] * scale
            p = torch.softmax(s, 0)
            out[b, h] = p @ v
            lse[b, h] = torch.logsumexp(s, 0) / math.log(2)
            e = (D + 8) * 2.0 ** -24 * float((k.abs() @ q[b, h].abs()).max()) * scale + 2.0 ** -22
            lse_bound[b, h] = 1.5 * e + 2.0 ** -23 * abs(float(lse[b, h])) + len(toks) * 2.0 ** -24 + 2.0 ** -20
            chain = (len(toks) / 32 + 64) * 2.0 ** -24
            bound[b, h] = half * out[b, h].abs() + (2 * e + chain) * (p @ v.abs()) + TINY[cache.key.dtype]
    return out, bound, lse, lse_bound


def check_decode(got, lse, ref):
    out, bound, l64, lb = ref
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(out))
    err = torch.nan_to_num((got - out).abs() / (bound + 1e-300))
    err[bound == 0] = (got - out).abs()[bound == 0]
    print(f"  out: worst error / bound {float(err.max()):.3f}", flush=True)
    assert float(err.max()) <= 1.0
    if lse is not None:
        lse = lse.double().cpu()
        dead = l64 == -math.inf
        assert bool((lse[dead] == -math.inf).all())
        assert bool(((lse - l64).abs()[~dead] <= lb[~dead]).all())


DECODE = [
    # dtype, H, Hkv, D, page, lengths, left, globals
    ("f32", 4, 4, 64, 16, [1, 15, 16, 17, 0, 200], None, 0),
    ("bf16", 8, 2, 128, 64, [64, 63, 65, 1, 700], None, 0),
    ("f16", 12, 4, 64, 32, [33, 2, 1000], None, 0),
    ("f16", 3, 1, 40, 48, [47, 49, 96], None, 0),
    ("bf16", 20, 1, 80, 16, [5, 300], None, 0),      # more than 16 queries on one key/value head
    ("f32", 33, 1, 128, 16, [129], None, 0),
    ("f32", 2, 2, 8, 16, [31, 32], None, 0),
    ("bf16", 4, 2, 16, 16, [0, 0], None, 0),
    ("f16", 8, 8, 64, 64, [500, 65, 64, 17, 3], 63, 0),
    ("bf16", 6, 3, 64, 16, [500, 65, 64, 17, 3, 1], 0, 0),
    ("f32", 4, 2, 48, 32, [333, 40, 17], 16, 20),    # globals that end inside a tile
    ("bf16", 8, 8, 64, 64, [2000, 100], 127, 16),
    ("bf16", 2, 2, 64, 16, [90], 1 << 40, 1 << 40),  # a window longer than any stream
    ("f16", 4, 2, 64, 1024, [1025, 1500, 1], None, 0),
]


def make_cache(pa, seed, dtype, pages, page, Hkv, D, B, width, lengths, sums=False):
    """A cache whose slots behind the lengths, and whose unused pages, hold NaN."""
    table = tables(seed, B, width, pages)
    k, v = (torch.full((pages, page, Hkv, D), float("nan"), dtype=dtype, device=DEV) for _ in range(2))
    for b, n in enumerate(lengths):
        for l in range((n + page - 1) // page):
            p, m = int(table[b, l]), min(page, n - l * page)
            k[p, :m], v[p, :m] = rnd(seed + 7 * b + 31 * l, 2, m, Hkv, D).to(dtype)
    return pa.PagedCache.from_tensors(k, v), table


@pytest.mark.parametrize("case", DECODE, ids=lambda c: f"{c[0]}-H{c[1]}.{c[2]}-D{c[3]}-p{c[4]}-w{c[6]}.{c[7]}")
def test_decode(pa, case):
    dt, H, Hkv, D, page, lengths, left, ng = case
    dtype, B = T[dt], len(lengths)
    width = max(1, (max(lengths) + page - 1) // page) + 1
    cache, table = make_cache(pa, 11, dtype, B * width + 2, page, Hkv, D, B, width, lengths)
    q = rnd(5, B, H, D, dtype=dtype)
    ref = decode64(q, cache, table, key_sets(lengths, Hkv, page, left, ng, None))
    got, lse = pa.paged_decode(q, cache, table, i32(*lengths), left=left, num_global=ng, return_lse=True)
    check_decode(got, lse, ref)
    assert same(got, pa.paged_decode(q, cache, table, i32(*lengths), left=left, num_global=ng))


@pytest.mark.parametrize("dt,page,D", [("bf16", 64, 64), ("f32", 16, 128), ("f16", 32, 32)])
def test_decode_listed_pages(pa, dt, page, D):
    """Lists with repeats, padding, pages behind the end, and nothing at all."""
    dtype, H, Hkv = T[dt], 8, 2
    lengths = [10 * page - 3, 3 * page + 1, 1, 0]
    B, width = 4, 10
    cache, table = make_cache(pa, 21, dtype, B * width, page, Hkv, D, B, width, lengths)
    pages = torch.tensor([[[9, 2, 2, 0, -1, 9], [5, 4, 3, 2, 1, 0]],
                          [[3, 7, -1, -9, 3, 1 << 30], [-1, -1, -1, -1, -1, -1]],
                          [[0, 0, 0, 0, 0, 0], [1, 2, 3, 4, 5, 6]],
                          [[0, 1, -1, -1, -1, -1], [0, 0, 0, 0, 0, 0]]], dtype=torch.int32, device=DEV)
    q = rnd(5, B, H, D, dtype=dtype)
    ref = decode64(q, cache, table, key_sets(lengths, Hkv, page, None, 0, pages.cpu()))
    got, lse = pa.paged_decode(q, cache, table, i32(*lengths), pages=pages, return_lse=True)
    check_decode(got, lse, ref)


def test_decode_bad_table_entries_are_skipped(pa):
    lengths, page = [100, 60], 16
    cache, table = make_cache(pa, 31, torch.float32, 20, page, 2, 32, 2, 7, lengths)
    table[0, 2], table[0, 4], table[1, 0], table[1, 1] = -1, 20, 1 << 30, -(1 << 31)
    q = rnd(5, 2, 4, 32)
    ref = decode64(q, cache, table, key_sets(lengths, 2, page, None, 0, None))
    got, lse = pa.paged_decode(q, cache, table, i32(*lengths), return_lse=True)
    check_decode(got, lse, ref)
    # lengths outside the table are clamped to it
    clamped = pa.paged_decode(q, cache, table[:, :3].contiguous(), i32(1 << 30, -4))
    ref = decode64(q, cache, table, key_sets([48, 0], 2, page, None, 0, None))
    check_decode(clamped, None, ref)


@pytest.mark.parametrize("dt,H,Hkv,D,page,lengths,kw", [
    ("bf16", 8, 8, 64, 64, [20000], {}),
    ("f16", 4, 1, 128, 16, [9000, 513, 0, 1], {}),
    ("f32", 4, 2, 64, 32, [7777, 512], {}),
    ("f16", 2, 2, 64, 64, [30000], dict(left=15000, num_global=700)),
], ids=str)
def test_decode_split_over_the_length(pa, dt, H, Hkv, D, page, lengths, kw):
    dtype, B = T[dt], len(lengths)
    width = (max(lengths) + page - 1) // page
    pages = B * width + 1
    table = tables(3, B, width, pages)
    cache = pa.PagedCache.from_tensors(rnd(1, pages, page, Hkv, D, dtype=dtype), rnd(2, pages, page, Hkv, D, dtype=dtype))
    q = rnd(5, B, H, D, dtype=dtype, scale=2.0)
    ref = decode64(q, cache, table, key_sets(lengths, Hkv, page, kw.get("left"), kw.get("num_global", 0), None))
    got, lse = pa.paged_decode(q, cache, table, i32(*lengths), return_lse=True, **kw)
    check_decode(got, lse, ref)
    for _ in range(3):  # the split is fixed by the sizes: the same bits every time
        assert same(got, pa.paged_decode(q, cache, table, i32(*lengths), **kw))


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("lengths", [[40], [6000]], ids=["one_pass", "split"])
def test_decode_infinities(pa, dt, lengths):
    """An infinite score spoils its row as it does in a softmax; scores of -inf
    take no weight, and a row of nothing else is undefined."""
    dtype, page, n = T[dt], 16, lengths[0]
    width = (n + page - 1) // page
    table = tables(3, 1, width, width)
    mk = lambda s: rnd(s, width, page, 1, 32, dtype=dtype)  # noqa: E731
    q = torch.zeros(1, 1, 32, dtype=dtype, device=DEV)
    q[..., 0] = 1.0
    for bad, at in ((-math.inf, 3), (math.inf, 3), (-math.inf, slice(None)), (math.nan, 5)):
        k, v = mk(1), mk(2)
        k[:, :, 0, 0][:, at] = bad
        if bad != -math.inf:  # only one page, so that other rows of the split stay finite
            k[1:, :, 0, 0] = 0.25
        cache = pa.PagedCache.from_tensors(k, v)
        ref = decode64(q, cache, table, key_sets(lengths, 1, page, None, 0, None))
        if bool((k[:, :, 0, 0] == -math.inf).all()):
            ref = (ref[0] * math.nan, *ref[1:])
        got = pa.paged_decode(q, cache, table, i32(n))
        check_decode(got, None, ref)


def test_decode_scale_and_large_scores(pa):
    lengths, page = [77], 16
    cache, table = make_cache(pa, 41, torch.float16, 5, page, 2, 64, 1, 5, lengths)
    q = rnd(5, 1, 4, 64, dtype=torch.float16, scale=30.0)  # weights of one key
    sets = key_sets(lengths, 2, page, None, 0, None)
    for scale in (None, 0.5, 1e-3):
        check_decode(pa.paged_decode(q, cache, table, i32(77), scale=scale), None,
                     decode64(q, cache, table, sets, scale))


def test_offsets_past_32_bits(pa):
    """A cache of more than 2^31 elements: appended to and read at its far end."""
    Hkv, D, page, dtype = 8, 128, 64, torch.bfloat16
    pages = (1 << 31) // (Hkv * D * page) + 5
    cache = pa.PagedCache(pages, page, Hkv, D, dtype, DEV, key_sums=True)
    table = i32(pages - 1, 0, pages - 2).view(1, 3)
    n = 150
    k, v = rnd(1, 1, n, Hkv, D, dtype=dtype), rnd(2, 1, n, Hkv, D, dtype=dtype)
    pa.paged_append(cache, k, v, table, i32(0))
    q = rnd(3, 1, 8, D, dtype=dtype)
    got = pa.paged_decode(q, cache, table, i32(n))
    small = pa.PagedCache(3, page, Hkv, D, dtype, DEV, key_sums=True)
    t2 = i32(2, 0, 1).view(1, 3)
    pa.paged_append(small, k, v, t2, i32(0))
    assert same(got, pa.paged_decode(q, small, t2, i32(n)))
    for a, b in ((pages - 1, 2), (pages - 2, 1), (0, 0)):
        assert same(cache.key_sums[a], small.key_sums[b])
    assert same(pa.paged_select(q, cache, table, i32(n), 2), pa.paged_select(q, small, t2, i32(n), 2))


# ---------------------------------------------------------------- select

def select64(q, sums, table, lengths, page, S, first, local):
    q, sums, t = q.double().cpu(), sums.double().cpu(), table.cpu()
    B, H, D = q.shape
    Hkv = sums.shape[1]
    out = torch.full((B, Hkv, S), -1, dtype=torch.int32)
    for b, n in enumerate(lengths):
        np_ = (n + page - 1) // page
        for h in range(Hkv):
            qs = q[b].view(Hkv, -1, D)[h].sum(0)
            cand = []
            for l in range(np_):
                p = int(t[b, l])
                if not 0 <= p < sums.shape[0]:
                    continue
                s = float((sums[p, h] / page * qs).sum())
                s = -math.inf if math.isnan(s) else s
                forced = l < first or l >= np_ - local
                cand.append((not forced, -s, l))
            take = sorted(l for _, _, l in sorted(cand)[:S])
            out[b, h, :len(take)] = torch.tensor(take, dtype=torch.int32)
    return out


@pytest.mark.parametrize("dt,H,Hkv,D,page,lengths,S,first,local", [
    ("bf16", 8, 2, 64, 64, [64 * 300, 1000, 64, 1, 0], 16, 1, 1),
    ("f16", 4, 4, 128, 16, [16 * 700 + 1, 16 * 64], 64, 0, 1),
    ("f32", 3, 1, 40, 32, [32 * 9, 32 * 9 - 1], 8, 2, 3),
    ("bf16", 1, 1, 8, 16, [16 * 5000], 1, 0, 1),
    ("f32", 2, 2, 64, 16, [16 * 40, 16 * 3], 5, 5 - 1, 1),
], ids=str)
def test_select(pa, dt, H, Hkv, D, page, lengths, S, first, local):
    B, width = len(lengths), (max(lengths) + page - 1) // page
    pages = B * width
    table = tables(3, B, width, pages)
    sums = rnd(1, pages, Hkv, D, scale=8.0)
    cache = pa.PagedCache(pages, page, Hkv, D, T[dt], DEV)
    cache = pa.PagedCache.from_tensors(cache.key, cache.value, sums)
    q = rnd(2, B, H, D, dtype=T[dt])
    got = pa.paged_select(q, cache, table, i32(*lengths), S, first_pages=first, local_pages=local)
    assert torch.equal(got.cpu(), select64(q, sums, table, lengths, page, S, first, local))


def test_select_ties_and_bad_values(pa):
    """Equal scores go to the lower page, a zero query lists the first pages, NaN
    ranks last, infinities by their sign, bad table entries are never listed."""
    page, Hkv, D, width = 16, 1, 16, 600
    table = torch.arange(width, dtype=torch.int32, device=DEV).view(1, width)
    key = torch.zeros(width, page, Hkv, D, device=DEV)
    q = torch.zeros(1, 1, D, device=DEV)
    q[..., 0] = 1.0
    sums = torch.zeros(width, Hkv, D, device=DEV)
    sums[:, 0, 0] = torch.arange(width, device=DEV) // 100 % 3  # whole runs of ties
    sums[7, 0, 0], sums[9, 0, 0], sums[11, 0, 0] = math.inf, math.nan, -math.inf
    sums[20, 0, 1] = math.inf  # times 0: NaN
    lens = [width * page]
    cache = pa.PagedCache.from_tensors(key, key, sums)
    for qq in (q, -q, torch.zeros_like(q), q * 1e-30):
        for S in (1, 3, 40, 64):
            got = pa.paged_select(qq, cache, table, i32(*lens), S)
            assert torch.equal(got.cpu(), select64(qq, sums, table, lens, page, S, 0, 1)), S
    bad = table.clone()
    bad[0, 7], bad[0, 599], bad[0, 250] = -1, width, 1 << 30
    got = pa.paged_select(q, cache, bad, i32(*lens), 5)
    ref = select64(q, sums, bad, lens, page, 5, 0, 1)
    assert torch.equal(got.cpu(), ref) and 599 not in got.tolist()[0][0]
    # all scores NaN: the listed pages are still the lowest ones
    sums.fill_(math.nan)
    assert pa.paged_select(q, cache, table, i32(*lens), 3).tolist() == [[[0, 1, 599]]]


@pytest.mark.parametrize("width,length", [
    (1, 1), (40, 40), (64, 64), (65, 65), (200, 200), (256, 256), (257, 257), (512, 512), (513, 513), (513, 256),
    (513, 100), (1100, 1025), (4100, 4099),
])
@pytest.mark.parametrize("page", [16, 48])
def test_select_widths(pa, page, width, length):
    """Tables around the sizes where the kernel changes its selection and its
    workgroup, with runs of ties, NaN, infinities and pages of the table missing;
    pages of 48 tokens, whose quotients round."""
    Hkv, D, n = 2, 24, (length - 1) * page + 5
    g = torch.Generator().manual_seed(width + length + page)
    sums = torch.randint(-3, 4, (width, Hkv, D), generator=g).float()
    sums[torch.randint(0, width, (max(1, width // 9),), generator=g), 0, 3] = math.nan
    sums[torch.randint(0, width, (max(1, width // 9),), generator=g), 1, 5] = -math.inf
    table = torch.randperm(width, generator=g).to(torch.int32).view(1, width)
    table[0, ::7] = -1
    q = torch.zeros(1, 4, D)
    q[0, :, 3], q[0, 2, 5], q[0, 1, 4] = 1.0, 2.0, -0.5
    key = torch.zeros(width, page, Hkv, D, device=DEV)
    cache = pa.PagedCache.from_tensors(key, key, sums.to(DEV))
    for S in (1, 2, 7, 63, 64):
        got = pa.paged_select(q.to(DEV), cache, table.to(DEV), i32(n), S)
        assert torch.equal(got.cpu(), select64(q, sums, table, [n], page, S, 0, 1)), S


# ---------------------------------------------------------------- together

def plain_step(q, ks, vs, sel, page):
    """Attention of q [H, D] over the listed pages of keys/values [n, Hkv, D], float64."""
    n, Hkv, D = ks.shape
    H = q.shape[0]
    out = torch.zeros(H, D, dtype=torch.float64)
    for h in range(H):
        tok = torch.tensor([t for p in sel[h // (H // Hkv)] if p >= 0 for t in range(p * page, min(n, (p + 1) * page))])
        s = ks[tok, h // (H // Hkv)] @ q[h] * D ** -0.5
        out[h] = torch.softmax(s, 0) @ vs[tok, h // (H // Hkv)]
    return out


def test_prompt_then_tokens(pa):
    """A prompt of ragged streams, then single tokens: append, select, decode,
    against the whole sequence recomputed in 64 bits."""
    B, H, Hkv, D, page, S, dtype = 3, 4, 2, 64, 16, 4, torch.bfloat16
    prompt = [100, 37, 1]
    N, steps, width = max(prompt), 20, 8
    cache = pa.PagedCache(B * width, page, Hkv, D, dtype, DEV, key_sums=True)
    cache.key.fill_(float("nan"))
    cache.value.fill_(float("nan"))
    table = tables(1, B, width, B * width)
    rot = pa.Rotation(D, device=DEV)
    total = N + steps
    k, v, q = (rnd(s, B, total, h, D, dtype=dtype) for s, h in ((1, Hkv), (2, Hkv), (3, H)))
    length = i32(*prompt)
    pa.paged_append(cache, k[:, :N].contiguous(), v[:, :N].contiguous(), table, i32(0, 0, 0), counts=length, rotation=rot)
    own = [[(i, ) for i in range(n)] for n in prompt]  # which input row is a stream's t-th token
    for i in range(N, total):
        row = slice(i, i + 1)
        qr = pa.paged_append(cache, k[:, row].contiguous(), v[:, row].contiguous(), table, length, rotation=rot,
                             query=q[:, row].contiguous())[:, 0]
        length += 1
        pages = pa.paged_select(qr, cache, table, length, S, first_pages=1)
        got = pa.paged_decode(qr, cache, table, length, pages=pages)
        for b in range(B):
            own[b].append((i,))
        if i % 5:
            continue
        for b in range(B):
            rows = torch.tensor([x[0] for x in own[b]])
            n = len(rows)
            pos = torch.arange(n)[None]
            ks = rotate64(k[b:b + 1, rows.to(DEV)], pos, rot.inv_freq, False)[0].to(dtype).double()
            qs = rotate64(q[b:b + 1, row], pos[:, -1:], rot.inv_freq, False)[0, 0].to(dtype).double()
            vs = v[b, rows.to(DEV)].double().cpu()
            ref = plain_step(qs, ks, vs, pages[b].tolist(), page)
            err = (got[b].double().cpu() - ref).abs()
            assert bool((err <= 2.0 ** -8 * ref.abs() + 1e-4).all()), (i, b, float(err.max()))
            sums = torch.stack([x.sum(0) for x in ks.split(page)])
            want = select64(qs[None], sums, torch.arange(len(sums))[None], [n], page, S, 1, 1)
            assert torch.equal(pages[b].cpu(), want[0]), (i, b)


def test_graph_replays(pa):
    """A decode step (append, select, decode with a split) in a graph: replays with
    new inputs equal the eager calls, with eager work in between; two graphs of the
    same step replayed in turn."""
    B, H, Hkv, D, page, width, dtype = 2, 4, 2, 64, 64, 80, torch.float16
    pages = B * width
    table = tables(1, B, width, pages)
    rot = pa.Rotation(D, device=DEV)

    def fresh():
        return pa.PagedCache.from_tensors(rnd(1, pages, page, Hkv, D, dtype=dtype), rnd(2, pages, page, Hkv, D, dtype=dtype),
                                          rnd(3, pages, Hkv, D))

    def step(cache, q, k, v, length):
        qr = pa.paged_append(cache, k, v, table, length, rotation=rot, query=q)[:, 0]
        sel = pa.paged_select(qr, cache, table, length + 1, 8)
        return pa.paged_decode(qr, cache, table, length + 1, pages=sel), pa.paged_decode(qr, cache, table, length + 1)

    bufs = [rnd(9, B, 1, h, D, dtype=dtype) for h in (H, Hkv, Hkv)]
    length = i32(4500, 77)
    captured, eager = fresh(), fresh()
    step(fresh(), *bufs, length)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(captured, *bufs, length)
        graphs.append((g, out))
    for r in range(6):
        for i, h in enumerate((H, Hkv, Hkv)):
            bufs[i].copy_(rnd(100 + 3 * r + i, B, 1, h, D, dtype=dtype))
        length += 1
        g, out = graphs[r % 2]
        g.replay()
        ref = step(eager, *bufs, length)
        torch.cuda.synchronize()
        assert same(out[0], ref[0]) and same(out[1], ref[1]), r
        assert same(captured.key, eager.key) and same(captured.key_sums, eager.key_sums), r


def test_other_stream_and_events(pa):
    import sparse_attention_cuda as ext
    cache, table = make_cache(pa, 51, torch.bfloat16, 300, 16, 2, 64, 2, 140, [2000, 1500])
    q = rnd(5, 2, 4, 64, dtype=torch.bfloat16)
    n = i32(2000, 1500)
    ref = pa.paged_decode(q, cache, table, n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = pa.paged_decode(q, cache, table, n)
    torch.cuda.current_stream().wait_stream(side)
    assert same(got, ref)
    e = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
    for x in e:
        x.record()
    torch.cuda.synchronize()
    with ext.kernel_events(*e):
        got = pa.paged_decode(q, cache, table, n)
    torch.cuda.synchronize()
    assert same(got, ref) and 0.0 < e[0].elapsed_time(e[1]) < 100.0


def test_refusals(pa):
    cache = pa.PagedCache(4, 16, 2, 64, torch.bfloat16, DEV)
    t, n = i32(0, 1).view(1, 2), i32(5)
    q = rnd(1, 1, 4, 64, dtype=torch.bfloat16)
    kv = rnd(1, 1, 3, 2, 64, dtype=torch.bfloat16)
    bad = [
        (lambda: pa.paged_decode(q.float(), cache, t, n), "torch.bfloat16"),
        (lambda: pa.paged_decode(q[:, :3].contiguous(), cache, t, n), "multiple"),
        (lambda: pa.paged_decode(q.transpose(1, 2), cache, t, n), "head_dim|contiguous"),
        (lambda: pa.paged_decode(q[..., :32], cache, t, n), "contiguous"),
        (lambda: pa.paged_decode(q, cache, t.long(), n), "int32"),
        (lambda: pa.paged_decode(q, cache, t, n.cpu()), "device tensor"),
        (lambda: pa.paged_decode(q, cache, t, i32(1, 2)), "shape"),
        (lambda: pa.paged_decode(q, cache, t.expand(3, 2).contiguous(), n), "row per stream"),
        (lambda: pa.paged_decode(q, cache, t, n, left=-1), "left"),
        (lambda: pa.paged_decode(q, cache, t, n, num_global=3), "num_global"),
        (lambda: pa.paged_decode(q, cache, t, n, pages=i32(0).view(1, 1, 1)), "pages must be"),
        (lambda: pa.paged_decode(q, cache, t, n, left=3, pages=i32(0, 0).view(1, 2, 1)), "exclude"),
        (lambda: pa.paged_decode(q, cache, t, n, scale=0.0), "scale"),
        (lambda: pa.paged_select(q, cache, t, n, 4), "key_sums"),
        (lambda: pa.paged_append(cache, kv, kv.float(), t, n), "value must be"),
        (lambda: pa.paged_append(cache, kv[..., :1, :].contiguous(), kv, t, n), "as the cache"),
        (lambda: pa.paged_append(cache, kv, kv, t, n, counts=n.long()), "int32"),
        (lambda: pa.paged_append(cache, kv, kv, t, n, rotation=pa.Rotation(128, device=DEV)), "exceeds"),
        (lambda: pa.paged_append(cache, kv, kv, t, n, rotation=pa.Rotation(64, device="cpu")), "another device"),
        (lambda: pa.paged_append(cache, kv, kv, t, n, query=q), "dimensions"),
        (lambda: pa.PagedCache(4, 20, 2, 64, torch.bfloat16, DEV), "page_size"),
        (lambda: pa.PagedCache(4, 16, 2, 60, torch.bfloat16, DEV), "head_dim"),
        (lambda: pa.PagedCache(4, 16, 2, 64, torch.float64, DEV), "dtype"),
    ]
    import re
    for call, msg in bad:
        with pytest.raises(RuntimeError) as e:
            call()
        assert re.search(msg, str(e.value)), (msg, str(e.value))
    # not 16-byte aligned
    flat = torch.zeros(4 * 64 + 1, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="aligned"):
        pa.paged_decode(flat[1:].view(1, 4, 64), cache, t, n)
