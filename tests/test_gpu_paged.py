"""Paged key / value caches on the device (nst_paged_plan, nst_paged_append, nst_paged_attention, nst_paged_reorder) against the float64
restatement of their contracts (oracle/kernel_emulation.py) at the sizes where they can go wrong: empty requests, one token, pages that
end inside every tile, heads of odd sizes, strided operands, entries outside their range, full pools.

Tolerances.  Everything that only moves data or counts is compared for equality.  The attention sums n terms in f32 (u = 2^-24): a score
is off by at most u (dh + 4) scale sum|q||k| (products and sum) + 3 u |s| (scale and log2 e), which scales a weight by twice that; the two
sums add at most 2 (n + 8) u.  With bf16 a weight is the sum of two roundings (off by 2^-8 of 2^-8 of itself) and the output is rounded
(2^-8 of itself):
    |o - o64| <= [2 ds + 2 (n + 8) u] sum p|v|   +   bf16: 2^-16 sum p|v| + 2^-8 |o64|,   f32: u |o64|
"""
import math

import pytest
import torch

from oracle import kernel_emulation as E

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24


@pytest.fixture(scope="module")
def K():
    from neurst_amd import kernels
    return kernels


def i32(a):
    return torch.tensor(a, dtype=torch.int32)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def make_cache(lens, ps, Hk, dh, dtype, seed, layout="token", spare_pages=3, width=None):
    """(k_pool, v_pool, table, lens) on the host: pages in random order, NaN wherever no token of a request lives."""
    g = gen(seed)
    held = [-(-n // ps) for n in lens]
    P = sum(held) + spare_pages
    order = torch.randperm(P, generator=g).tolist()
    W = width or max(held + [1])
    table = torch.full((len(lens), W), -1, dtype=torch.int32)
    shape = (P, ps, Hk, dh) if layout == "token" else (P, Hk, ps, dh)
    pools = [torch.full(shape, float("nan")).to(dtype) for _ in range(2)]
    views = [p if layout == "token" else p.transpose(1, 2) for p in pools]
    at = 0
    for b, n in enumerate(lens):
        for j in range(held[b]):
            page = order[at]
            at += 1
            table[b, j] = page
            rows = min(ps, n - j * ps)
            for p in views:
                p[page, :rows] = torch.randn(rows, Hk, dh, generator=g).to(dtype)
    return views[0], views[1], table, i32(lens)


def attention_reference(q, k_pool, v_pool, table, lens, scale):
    """out, lse and the tolerance of out, float64."""
    B, H, dh = q.shape
    P, ps, Hk = k_pool.shape[:3]
    out, lse, tol = (torch.zeros(B, H, dh, dtype=torch.float64), torch.full((B, H), -math.inf, dtype=torch.float64),
                     torch.zeros(B, H, dh, dtype=torch.float64))
    half = 2.0 ** -8 if q.dtype == torch.bfloat16 else 0.0
    for b in range(B):
        n = min(max(int(lens[b]), 0), table.shape[1] * ps)
        t = torch.arange(n)
        page = table[b].long()[t // ps] if n else t
        keep = (page >= 0) & (page < P)
        page, off = page[keep], (t % ps)[keep]
        if page.numel() == 0:
            continue
        k, v = k_pool[page, off].double(), v_pool[page, off].double()
        for h in range(H):
            kh, vh, qh = k[:, h // (H // Hk)], v[:, h // (H // Hk)], q[b, h].double()
            s = kh @ qh * scale
            p = torch.softmax(s, 0)
            ds = float((U * (dh + 4) * abs(scale) * (kh.abs() @ qh.abs()) + 3 * U * s.abs()).max())
            mag = p @ vh.abs()
            out[b, h], lse[b, h] = p @ vh, torch.logsumexp(s, 0)
            tol[b, h] = (2 * ds + 2 * (page.numel() + 8) * U + half * half) * mag + max(half, U) * out[b, h].abs()
    return out, lse, tol


def run_attention(K, q, k_pool, v_pool, table, lens, scale=None, **kw):
    dh = q.shape[2]
    want, want_lse, tol = attention_reference(q, k_pool, v_pool, table, lens, dh ** -0.5 if scale is None else scale)
    d = lambda t: t.to(DEV)     # noqa: E731
    kd, vd = to_device_like(k_pool), to_device_like(v_pool)
    out, lse = K.paged_attention(d(q), kd, vd, d(table), d(lens), scale=scale, return_lse=True, **kw)
    assert out.dtype == q.dtype and out.shape == q.shape and lse.dtype == torch.float32
    err = (out.cpu().double() - want).abs()
    assert torch.isfinite(out).all()
    assert (err <= tol + 1e-30).all(), f"worst {float((err / (tol + 1e-30)).max()):.2f} of the tolerance"
    empty = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse.cpu()), empty) and (out.cpu()[empty] == 0).all()
    # lse: the scores' error, the sum's, and the rounding of the result itself
    e = (lse.cpu().double() - want_lse)[~empty].abs()
    if e.numel():
        n = int(lens.max())
        ds = 4 * U * (dh + 8) * 8.0 * math.sqrt(dh) * (1 if scale is None else abs(scale) * math.sqrt(dh))
        assert float(e.max()) <= ds + (n + 16) * U + 4 * U * float(want_lse[~empty].abs().max()), float(e.max())
    return out


def to_device_like(t):
    """The same strides on the device (a transposed pool stays transposed)."""
    base = torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=DEV)
    base.copy_(t)
    return base


# ------------------------------------------------------------------------------------------------ attention
LENS = {"mixed": [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 257], "one": [1], "none": [0], "long": [2049, 7, 0, 513]}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("ps", [1, 7, 16, 24, 64])
@pytest.mark.parametrize("which", sorted(LENS))
def test_attention_over_lengths_and_page_sizes(K, which, ps, dtype):
    lens = LENS[which]
    k, v, table, ln = make_cache(lens, ps, 2, 64, dtype, seed=ps)
    q = torch.randn(len(lens), 4, 64, generator=gen(1)).to(dtype)
    run_attention(K, q, k, v, table, ln)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,Hk,dh", [(1, 1, 1), (1, 1, 8), (2, 1, 5), (4, 4, 32), (6, 2, 40), (8, 1, 64), (4, 2, 80), (3, 3, 96), (5, 1, 128),
                                     (32, 2, 128), (40, 2, 64), (2, 1, 200), (2, 2, 256), (17, 1, 33)])
def test_attention_over_heads_and_head_sizes(K, H, Hk, dh, dtype):
    lens = [70, 0, 33, 129, 5]
    k, v, table, ln = make_cache(lens, 16, Hk, dh, dtype, seed=dh)
    q = torch.randn(len(lens), H, dh, generator=gen(H)).to(dtype)
    run_attention(K, q, k, v, table, ln)
    run_attention(K, q, k, v, table, ln, scale=0.3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("max_len", [None, 1, 64, 100000])
def test_the_bound_of_the_lengths_never_changes_the_extent(K, max_len, dtype):
    lens = [1500, 3, 700, 0, 64]
    k, v, table, ln = make_cache(lens, 32, 2, 64, dtype, seed=3, width=60)
    q = torch.randn(len(lens), 4, 64, generator=gen(2)).to(dtype)
    run_attention(K, q, k, v, table, ln, max_len=max_len)


@pytest.mark.parametrize("B,lens_hi", [(1, 5000), (3, 9000), (300, 300)])
def test_attention_split_over_the_length_and_over_many_requests(K, B, lens_hi):
    lens = [(lens_hi * (i + 1)) // B for i in range(B)]
    k, v, table, ln = make_cache(lens, 16, 1, 64, torch.bfloat16, seed=B)
    q = torch.randn(B, 2, 64, generator=gen(2)).to(torch.bfloat16)
    run_attention(K, q, k, v, table, ln)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dh", [1, 20, 40, 64, 100, 128, 200, 256])
@pytest.mark.parametrize("max_len", [600, 5000])
def test_attention_joins_parts_of_every_head_size(K, max_len, dh, dtype):
    """3 and 20 parts at most: both forms of the join, and requests that fill one part or none of them."""
    lens = [600, 0, 5, 257, 128, 513]
    k, v, table, ln = make_cache(lens, 16, 2, dh, dtype, seed=dh, width=max_len // 16 + 1)
    q = torch.randn(len(lens), 6, dh, generator=gen(2)).to(dtype)
    run_attention(K, q, k, v, table, ln, max_len=max_len)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_reads_strided_operands(K, dtype):
    lens = [50, 17, 0, 90]
    H, Hk, dh = 4, 2, 48
    k, v, table, ln = make_cache(lens, 8, Hk, dh, dtype, seed=9, layout="head")       # [pages, heads, page_size, dh]
    packed = torch.randn(len(lens), 3, H * dh, generator=gen(4)).to(dtype)
    q = packed[:, 1].view(len(lens), H, dh)
    assert not k.is_contiguous() and not q.is_contiguous()
    want, _, tol = attention_reference(q, k, v, table, ln, dh ** -0.5)
    wide = torch.full((len(lens), table.shape[1] + 5), -7, dtype=torch.int32)
    wide[:, 2:2 + table.shape[1]] = table
    wd = wide.to(DEV)
    out = K.paged_attention(packed.to(DEV)[:, 1].view(len(lens), H, dh), to_device_like(k), to_device_like(v), wd[:, 2:2 + table.shape[1]],
                            ln.to(DEV))
    assert ((out.cpu().double() - want).abs() <= tol + 1e-30).all()
    # a pool that starts one element behind an aligned address
    flat = torch.empty(k.numel() * 2 + 1, dtype=dtype, device=DEV)
    n = k.numel()
    ku, vu = (flat[1 + i * n:1 + (i + 1) * n].view(k.shape) for i in range(2))
    ku.copy_(k), vu.copy_(v)
    out2 = K.paged_attention(q.to(DEV), ku, vu, table.to(DEV), ln.to(DEV))
    assert ((out2.cpu().double() - want).abs() <= tol + 1e-30).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_ignores_pages_outside_the_pool_and_lengths_outside_the_table(K, dtype):
    lens = [100, 64, 40, 16, 90, 10]
    k, v, table, ln = make_cache(lens, 16, 2, 64, dtype, seed=5)
    P = k.shape[0]
    table[0, 2], table[1, 0], table[1, 3], table[3, 0] = P, -5, 2 ** 31 - 1, -1        # request 3 keeps nothing
    ln = i32([100, 64, 40, 16, 10 ** 9, -3])
    q = torch.randn(len(lens), 4, 64, generator=gen(6)).to(dtype)
    # request 4 claims more tokens than its table row reaches: the row is read to its end (its last page holds unset rows)
    tail = table.shape[1] * 16
    for pool in (k, v):
        for t in range(90, tail):
            page = int(table[4, t // 16])
            if 0 <= page < P:
                pool[page, t % 16] = 0.25
    run_attention(K, q, k, v, table, ln)


def test_attention_of_large_scores_and_infinities(K):
    """The running maximum: scores around +-1e4, one key that takes everything, a minus infinity among the keys."""
    lens = [200, 200, 40]
    k, v, table, ln = make_cache(lens, 16, 1, 64, torch.float32, seed=7)
    q = torch.randn(3, 1, 64, generator=gen(6))
    q[0] *= 1000.0
    page = int(table[1, 150 // 16])
    k[page, 150 % 16] = q[1] * 50
    run_attention(K, q, k, v, table, ln)
    q[2] = 1.0
    page = int(table[2, 1])
    k[page, 3, 0, 0] = -math.inf                               # score -inf: weight exactly 0
    out = K.paged_attention(q.to(DEV), k.to(DEV), v.to(DEV), table.to(DEV), ln.to(DEV)).cpu()
    pos = [t for t in range(40) if t != 19]
    kk = torch.stack([k[int(table[2, t // 16]), t % 16, 0] for t in pos]).double()
    vv = torch.stack([v[int(table[2, t // 16]), t % 16, 0] for t in pos]).double()
    want = torch.softmax(kk.sum(1) / 8.0, 0) @ vv
    assert float((out[2, 0].double() - want).abs().max()) < 1e-4


def test_attention_past_32_bit_offsets(K):
    """A pool whose later pages lie more than 2^31 elements behind its start (built as a view with a wide page stride)."""
    dh, ps, P = 64, 16, 5
    stride = 2 ** 29 + 2 ** 27                                  # elements between pages: page 4 starts 5 GiB into the bf16 buffer
    flat = torch.zeros(stride * (P - 1) + ps * dh, dtype=torch.bfloat16, device=DEV)
    k = torch.as_strided(flat, (P, ps, 1, dh), (stride, dh, dh, 1))
    rows = torch.randn(P, ps, 1, dh, generator=gen(0)).to(torch.bfloat16)
    k.copy_(rows)
    table, ln = i32([[4, 1, 3, 0, 2]]), i32([75])
    q = torch.randn(1, 1, dh, generator=gen(1)).to(torch.bfloat16)
    want, _, tol = attention_reference(q, rows, rows, table, ln, dh ** -0.5)
    out = K.paged_attention(q.to(DEV), k, k, table.to(DEV), ln.to(DEV))
    assert ((out.cpu().double() - want).abs() <= tol).all()
    k2 = torch.as_strided(flat, (P, ps, 1, dh), (stride, dh, dh, 1))
    new = torch.randn(2, 1, dh, generator=gen(3)).to(torch.bfloat16)
    K.paged_append(new.to(DEV), new.to(DEV), k2, k2, torch.tensor([4 * ps + 3, 2 * ps], device=DEV))
    assert torch.equal(k2[4, 3].cpu(), new[0]) and torch.equal(k2[2, 0].cpu(), new[1])


# ------------------------------------------------------------------------------------------------ plan
@pytest.mark.parametrize("ps", [1, 5, 16, 64])
@pytest.mark.parametrize("B,cached_hi,new_hi", [(1, 0, 1), (1, 40, 5000), (7, 30, 3), (256, 100, 1), (257, 70, 40), (1000, 20, 0), (3000, 50, 9)])
def test_plan_matches_its_contract(K, B, cached_hi, new_hi, ps):
    g = gen(B + ps)
    cached = torch.randint(0, cached_hi + 1, (B,), generator=g).int()
    new = torch.randint(0, new_hi + 1, (B,), generator=g).int()
    held = (cached + ps - 1) // ps
    W = int(((cached + new + ps - 1) // ps).max()) + 2
    pages = torch.randperm(int(((cached + new + ps - 1) // ps).sum()) + 9, generator=g).int()
    table = torch.full((B, W + 3), -1, dtype=torch.int32)[:, 1:W + 1]
    at = 0
    for b in range(B):
        table[b, :held[b]] = pages[at:at + int(held[b])]
        at += int(held[b])
    free, cursor = pages[at:].contiguous(), i32([4])
    total = int(new.sum())
    for extra in (0, 13, -(total // 3)):          # (the last: fewer slots than tokens)
        t_ref = table.clone()
        t_dev = torch.full((B, W + 3), -1, dtype=torch.int32, device=DEV)[:, 1:W + 1]
        t_dev.copy_(table)
        want = E.paged_plan(cached, new, t_ref, free, cursor, ps, total + extra)
        got = K.paged_plan(cached.to(DEV), new.to(DEV), t_dev, free.to(DEV), cursor.to(DEV), ps, total + extra)
        for a, b in zip(got, want):
            assert a.dtype == b.dtype and torch.equal(a.cpu(), b)
        assert torch.equal(t_dev.cpu(), t_ref)


@pytest.mark.parametrize("n_free,cursor", [(0, 0), (3, 0), (3, 3), (3, 50), (5, 2)])
def test_plan_with_too_few_pages_and_full_table_rows(K, n_free, cursor):
    """Requests are served in order; tokens without a page get slot -1 and are not counted; a row of the table that is full takes no more."""
    cached, new = i32([3, 8, 0, 16, 5, -2, 1000]), i32([4, 9, -3, 6, 2, 3, 5])
    ps, W = 4, 5
    table = torch.arange(100, 100 + 7 * W, dtype=torch.int32).view(7, W)
    for b in range(7):
        table[b, -(-min(max(int(cached[b]), 0), W * ps) // ps):] = -1
    free = torch.arange(n_free, dtype=torch.int32) + 50
    t_ref, t_dev = table.clone(), table.to(DEV)
    want = E.paged_plan(cached, new, t_ref, free, i32([cursor]), ps, 40)
    got = K.paged_plan(cached.to(DEV), new.to(DEV), t_dev, free.to(DEV), i32([cursor]).to(DEV), ps, 40)
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b), (a.cpu(), b)
    assert torch.equal(t_dev.cpu(), t_ref)


def test_plan_with_senseless_lengths_ends(K):
    """Lengths near 2^31 in every request, pages of one token in a table row of 2^20: what cannot be served costs nothing."""
    B, W = 70, 1 << 20
    big = 2 ** 31 - 1
    cached, new = i32([big, -big - 1, 5] + [0] * (B - 3)), i32([big] * B)
    table = torch.full((B, W), -1, dtype=torch.int32, device=DEV)
    slots, lens, cu, cursor = K.paged_plan(cached.to(DEV), new.to(DEV), table, torch.arange(9, dtype=torch.int32, device=DEV), i32([4]).to(DEV), 1, 20)
    # request 0 is full; the five free pages go to request 1, whose tokens stand behind request 0's and past the twenty slots
    assert slots.tolist() == [-1] * 20 and cursor.tolist() == [9] and lens.tolist() == [W, 0, 5] + [0] * (B - 3)
    assert table[1, :6].tolist() == [4, 5, 6, 7, 8, -1]


# ------------------------------------------------------------------------------------------------ append
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,Hk,dh,ps", [(1, 1, 1, 1), (5, 2, 5, 3), (128, 4, 64, 16), (1000, 8, 40, 24), (333, 1, 256, 7)])
def test_append_writes_its_slots_and_nothing_else(K, T, Hk, dh, ps, dtype):
    g = gen(T)
    P = -(-T // ps) + 2
    qkv = torch.randn(T, 3, Hk * dh, generator=g).to(dtype)
    pool = torch.randn(2, P, ps, Hk, dh, generator=g).to(dtype)
    slots = torch.randperm(P * ps, generator=g)[:T]
    if T > 4:
        slots[1], slots[2], slots[3] = -1, P * ps, -2 ** 62
    kr, vr = pool[0].clone(), pool[1].clone()
    k, v = qkv[:, 1].view(T, Hk, dh), qkv[:, 2].view(T, Hk, dh)
    E.paged_append(k, v, kr, vr, slots)
    qd, pd = qkv.to(DEV), pool.to(DEV)
    K.paged_append(qd[:, 1].view(T, Hk, dh), qd[:, 2].view(T, Hk, dh), pd[0], pd[1], slots.to(DEV))
    assert torch.equal(pd[0].cpu(), kr) and torch.equal(pd[1].cpu(), vr)
    # heads in front of tokens in a page
    alt = torch.zeros(2, P, Hk, ps, dh, dtype=dtype, device=DEV)
    K.paged_append(qd[:, 1].view(T, Hk, dh), qd[:, 2].view(T, Hk, dh), alt[0].transpose(1, 2), alt[1].transpose(1, 2), slots.to(DEV))
    zero = torch.zeros(2, P, ps, Hk, dh, dtype=dtype)
    E.paged_append(k, v, zero[0], zero[1], slots)
    assert torch.equal(alt.transpose(2, 3).cpu(), zero)


# ------------------------------------------------------------------------------------------------ reorder
def reorder_case(groups, beam, N, C, ps, dtype, lens, seed):
    g = gen(seed)
    R = groups * beam
    ln = i32([n for n in lens for _ in range(beam)])
    held = [-(-int(n) // ps) for n in ln]
    W = max(held) + 2
    pages = torch.randperm(sum(held) + R + 2, generator=g).int()
    table = torch.full((R, W), -1, dtype=torch.int32)
    at = 0
    for r in range(R):
        table[r, :held[r]] = pages[at:at + held[r]]
        at += held[r]
    spare = pages[at:at + R].clone()
    parents = torch.tensor([(r // beam) * beam + int(torch.randint(0, beam, (1,), generator=g)) for r in range(R)])
    pool = torch.randn(N, pages.numel(), ps, C, generator=g).to(dtype)
    return pool, table, ln, parents, spare


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("groups,beam,N,C,ps,lens", [(1, 1, 1, 1, 1, [3]), (3, 4, 4, 64, 16, [1, 16, 75]), (2, 5, 3, 33, 7, [0, 20]),
                                                     (5, 2, 2, 256, 8, [9, 8, 7, 1, 31]), (40, 3, 6, 40, 4, [5] * 40)])
def test_reorder_matches_its_contract(K, groups, beam, N, C, ps, lens, dtype):
    pool, table, ln, parents, spare = reorder_case(groups, beam, N, C, ps, dtype, lens, seed=beam + C)
    if table.shape[0] > 4:      # rows that keep their own sequence: no such parent, a parent of another length, no such spare page
        parents[0], parents[1], spare[2] = -1, table.shape[0], -9
        if len(set(lens)) > 1:
            parents[3] = table.shape[0] - 1
    ref = pool.clone()
    want = E.paged_reorder(ref, table, ln, parents, spare)
    pd = pool.to(DEV)
    got = K.paged_reorder(pd, table.to(DEV), ln.to(DEV), parents.to(DEV), spare.to(DEV))
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
    assert torch.equal(pd.cpu(), ref)


# ------------------------------------------------------------------------------------------------ as they are used
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_run_of_steps_equals_a_dense_cache(K, dtype):
    """Plan, append, attend and re-order over several steps of a beam search, ragged prompts first, against dense per-row histories."""
    torch.manual_seed(0)
    R, beam, Hk, H, dh, ps, W, steps = 12, 3, 2, 4, 32, 4, 8, 9
    P = R * (W + 1)
    g = gen(12)
    pool = torch.zeros(2, P, ps, Hk * dh, dtype=dtype, device=DEV)
    kp, vp = pool[0].view(P, ps, Hk, dh), pool[1].view(P, ps, Hk, dh)
    ring = torch.randperm(P, generator=g).int()
    spare, free = ring[:R].to(DEV), ring[R:].contiguous().to(DEV)
    cursor = torch.zeros(1, dtype=torch.int32, device=DEV)
    table = torch.full((R, W), -1, dtype=torch.int32, device=DEV)
    lens = torch.zeros(R, dtype=torch.int32, device=DEV)
    hist = [([], []) for _ in range(R)]
    prompt = [1 + (r // beam) * 3 for r in range(R)]
    for step in range(steps):
        new = prompt if step == 0 else [1] * R
        T = sum(new)
        slots, lens, cu, cursor = K.paged_plan(lens, i32(new).to(DEV), table, free, cursor, ps, T + 2)
        kv = torch.randn(T + 2, 2, Hk * dh, generator=g).to(dtype)
        kd = kv.to(DEV)
        K.paged_append(kd[:, 0].view(T + 2, Hk, dh), kd[:, 1].view(T + 2, Hk, dh), kp, vp, slots)
        cu = cu.cpu().tolist()
        for r in range(R):
            for t in range(cu[r], cu[r + 1]):
                hist[r][0].append(kv[t, 0].view(Hk, dh))
                hist[r][1].append(kv[t, 1].view(Hk, dh))
        q = torch.randn(R, H, dh, generator=g).to(dtype)
        out = K.paged_attention(q.to(DEV), kp, vp, table, lens, max_len=W * ps).cpu().double()
        assert lens.cpu().tolist() == [len(h[0]) for h in hist]
        for r in range(R):
            k, v = torch.stack(hist[r][0]), torch.stack(hist[r][1])
            n = k.shape[0]
            want, _, tol = attention_reference(q[r:r + 1], k[None], v[None], i32([[0]]), i32([n]), dh ** -0.5)
            assert ((out[r] - want[0]).abs() <= tol[0]).all(), (step, r)
        parents = torch.tensor([(r // beam) * beam + int(torch.randint(0, beam, (1,), generator=g)) for r in range(R)])
        table, spare = K.paged_reorder(pool, table, lens, parents.to(DEV), spare)
        hist = [(list(hist[p][0]), list(hist[p][1])) for p in parents.tolist()]


def test_captured_step_replays_with_new_lengths(K):
    """One captured graph of plan + append + attend serves every step: lengths, tables and cursors live on the device.  Two graphs captured
    on one stream have scratch of their own and may be replayed one after the other in any order."""
    R, Hk, H, dh, ps, W = 3, 1, 2, 64, 16, 200
    P = R * W
    g = gen(3)

    def make():
        return dict(kp=torch.zeros(P, ps, Hk, dh, dtype=torch.bfloat16, device=DEV), vp=torch.zeros(P, ps, Hk, dh, dtype=torch.bfloat16, device=DEV),
                    table=torch.full((R, W), -1, dtype=torch.int32, device=DEV), lens=torch.zeros(R, dtype=torch.int32, device=DEV),
                    cursor=torch.zeros(1, dtype=torch.int32, device=DEV), q=torch.zeros(R, H, dh, dtype=torch.bfloat16, device=DEV),
                    k=torch.zeros(R, Hk, dh, dtype=torch.bfloat16, device=DEV), v=torch.zeros(R, Hk, dh, dtype=torch.bfloat16, device=DEV))
    free, ones = torch.randperm(P, generator=g).int().to(DEV), torch.ones(R, dtype=torch.int32, device=DEV)

    def step(s):
        slots, lens, _, cursor = K.paged_plan(s["lens"], ones, s["table"], free, s["cursor"], ps, R)
        K.paged_append(s["k"], s["v"], s["kp"], s["vp"], slots)
        out = K.paged_attention(s["q"], s["kp"], s["vp"], s["table"], lens)
        s["lens"].copy_(lens)
        s["cursor"].copy_(cursor)
        return out
    states, graphs = [make(), make(), make()], []
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for s in states[:2]:
            step(s)                                                            # warm-up, undone below
            s["lens"].zero_(), s["cursor"].zero_(), s["table"].fill_(-1)
    torch.cuda.synchronize()
    for s in states[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = step(s)
        graphs.append((graph, out))
    for i in range(40):
        x = [torch.randn(R, n, dh, generator=g).to(torch.bfloat16).to(DEV) for n in (H, Hk, Hk)]
        for s in states:
            s["q"].copy_(x[0]), s["k"].copy_(x[1]), s["v"].copy_(x[2])
        order = (0, 1) if i % 2 else (1, 0)
        for n in order:
            graphs[n][0].replay()
        want = step(states[2])
        torch.cuda.synchronize()
        for n in range(2):
            assert torch.equal(graphs[n][1], want), i
            assert torch.equal(states[n]["lens"], states[2]["lens"]) and torch.equal(states[n]["table"], states[2]["table"])


def test_calls_on_another_stream(K):
    lens = [700, 30, 0]
    k, v, table, ln = make_cache(lens, 16, 2, 64, torch.bfloat16, seed=1)
    q = torch.randn(3, 4, 64, generator=gen(6)).to(torch.bfloat16).to(DEV)
    kd, vd, td, ld = k.to(DEV), v.to(DEV), table.to(DEV), ln.to(DEV)
    a = K.paged_attention(q, kd, vd, td, ld)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        b = K.paged_attention(q, kd, vd, td, ld)
    side.synchronize()
    assert torch.equal(a, b)


def test_calls_with_nothing_in_them(K):
    z = lambda *shape, dt=torch.int32: torch.zeros(*shape, dtype=dt, device=DEV)      # noqa: E731
    pool = z(4, 16, 2, 64, dt=torch.float32)
    assert K.paged_attention(z(0, 4, 64, dt=torch.float32), pool, pool, z(0, 3), z(0)).shape == (0, 4, 64)
    K.paged_append(z(0, 2, 64, dt=torch.float32), z(0, 2, 64, dt=torch.float32), pool, pool, z(0, dt=torch.int64))
    slots, lens, cu, cursor = K.paged_plan(z(0), z(0), z(0, 3), z(5), i32([2]).to(DEV), 16, 4)
    assert slots.tolist() == [-1] * 4 and lens.numel() == 0 and cu.tolist() == [0] and cursor.tolist() == [2]
    slots, lens, cu, cursor = K.paged_plan(i32([3, 0]).to(DEV), z(2), z(2, 3), z(0), z(1), 16, 0)
    assert slots.numel() == 0 and lens.tolist() == [3, 0] and cu.tolist() == [0, 0, 0] and cursor.tolist() == [0]
    t, s = K.paged_reorder(z(2, 4, 16, 8, dt=torch.float32), z(0, 3), z(0), z(0, dt=torch.int64), z(0))
    assert t.shape == (0, 3) and s.shape == (0,)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_over_a_pool_without_pages(K, dtype):
    """Nothing exists that a table could name: no row is read, every output is 0 -- whole requests and requests in parts."""
    pool = torch.zeros(0, 16, 2, 64, dtype=dtype, device=DEV)
    q = torch.randn(3, 4, 64, generator=gen(0)).to(dtype).to(DEV)
    for W in (2, 100):
        table = torch.zeros(3, W, dtype=torch.int32, device=DEV)
        out, lse = K.paged_attention(q, pool, pool, table, i32([W * 16, 5, 0]).to(DEV), return_lse=True)
        assert (out == 0).all() and torch.isinf(lse).all() and (lse < 0).all()


def test_two_calls_at_once(K):
    """Long requests on two streams at the same time: each call has scratch of its own."""
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    cases = []
    for i in range(2):
        k, v, table, ln = make_cache([3000, 4000 - 100 * i, 1], 16, 2, 64, torch.bfloat16, seed=i)
        q = torch.randn(3, 4, 64, generator=gen(6 + i)).to(torch.bfloat16)
        cases.append([t.to(DEV) for t in (q, k, v, table, ln)])
    want = [K.paged_attention(*c) for c in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(sides[i]):
                got[i].append(K.paged_attention(*cases[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_plan_with_entries_of_the_free_list_that_name_no_page(K):
    """They enter the table as -1, over whatever a row held there before: their tokens have no slot and attention does not see them."""
    table = i32([[3, 0, 7], [4, 6, 5], [1, 2, 0]])                                  # (stale entries behind each row's own pages)
    cached, new, free, cursor = i32([4, 0, 3]), i32([3, 9, 6]), i32([-5, 8, -1, 9, -2 ** 31, 10]), i32([0])
    want_table = table.clone()
    want = E.paged_plan(cached, new, want_table, free, cursor, 4, 20)
    td = table.to(DEV)
    got = K.paged_plan(cached.to(DEV), new.to(DEV), td, free.to(DEV), cursor.to(DEV), 4, 20)
    for g, w in zip(got, want):
        assert torch.equal(g.cpu(), w)
    assert torch.equal(td.cpu(), want_table) and want_table.tolist() == [[3, -1, 7], [8, -1, 9], [1, -1, 10]]
    k = torch.randn(11, 4, 1, 64, generator=gen(0))
    q = torch.randn(3, 2, 64, generator=gen(1))
    run_attention(K, q, k, k.flip(0).contiguous(), want_table, want[1])
