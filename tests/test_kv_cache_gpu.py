"""The paged key-value cache (append, single-token attention, key weights,
eviction) against plain forms in 64 bits.

Tolerances.  u = 2^-24 is half a step of fp32.  A score is a sum of D products in
fp32: off by at most e = (D + 4) u A, A the largest sum_d |q_d k_d| * scale (the
products of 16-bit inputs are exact, those of fp32 inputs rounded: the 4 covers
them, the scale and the exponent's argument).  A probability is then off by at
most a share of 2 e + (n + 8) u + 2^-20 (numerator and denominator, a sum of n
terms, the exponential's own 2 units in the last place on either side), and
16-bit probabilities are held as the sum of two 16-bit numbers: 2^-17 more.  An
output is a mean of V under them: off by that share of max |V|, and by half a
step of its own type, eps / 2 of the value.  The log-sum-exp is off by that
share plus its own rounding."""
import ctypes
import math
import threading

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _pools(P, H, page, D, dtype, g, layout="heads"):
    """Two pools of random rows; layout "slots": [P, page, H, D] in memory."""
    shape = (P, H, page, D) if layout == "heads" else (P, page, H, D)
    mk = lambda: torch.randn(shape, device="cuda", generator=g).to(dtype)  # noqa: E731
    k, v = mk(), mk()
    return (k, v) if layout == "heads" else (k.transpose(1, 2), v.transpose(1, 2))


def _table(B, M, P, g):
    return torch.randperm(P, device="cuda", generator=g)[: B * M].to(torch.int32).view(B, M)


def _rows(k, v, table, b, n):
    """Positions, keys and values of sequence b's first n positions that a page holds, in 64 bits."""
    page, P = k.shape[2], k.shape[0]
    pos = torch.arange(max(0, min(n, table.shape[1] * page)), device="cuda")
    pg = table[b].long()[pos // page] if pos.numel() else pos
    there = (pg >= 0) & (pg < P)
    pos, pg = pos[there], pg[there]
    return pos, k[pg, :, pos % page].double(), v[pg, :, pos % page].double()  # [n, H, D]


def _check_attention(gae, q, k, v, table, lens, scale=None, weights=None, got=None, **kw):
    B, H, D = q.shape
    Hkv = k.shape[1]
    G = H // Hkv
    sc = 1 / math.sqrt(D) if scale is None else scale
    w_in = None if weights is None else weights.clone()
    if got is None:
        got = gae.paged_attention(q, k, v, table, lens, scale=scale, return_lse=True, weights=weights, **kw)
    out, lse = got
    torch.cuda.synchronize()
    gae.device_status()
    w_out = kw.get("weights_out", weights)
    half = torch.finfo(q.dtype).eps / 2
    for b, n in enumerate(lens.tolist()):
        pos, kb, vb = _rows(k, v, table, b, n)
        if pos.numel() == 0:
            assert (out[b] == 0).all() and (lse[b] == -math.inf).all()
            if weights is not None:
                assert torch.equal(w_out[b], w_in[b])
            continue
        if weights is not None:
            rest = torch.ones(w_out.shape[2], dtype=torch.bool, device="cuda")
            rest[pos] = False
            assert torch.equal(w_out[b][:, rest], w_in[b][:, rest])
        for j in range(Hkv):
            qg = q[b, j * G: (j + 1) * G].double()
            x = qg @ kb[:, j].T * sc
            A = (qg.abs() @ kb[:, j].abs().T * sc).max().item()
            share = 2 * (D + 4) * U * A + (len(pos) + 8) * U + 2.0 ** -20 + (2.0 ** -17 if q.dtype != torch.float32 else 0)
            p = torch.softmax(x, 1)
            ref = p @ vb[:, j]
            err = (out[b, j * G: (j + 1) * G].double() - ref).abs()
            assert (err <= half * ref.abs() + share * vb[:, j].abs().max()).all(), (b, j, err.max().item())
            rl = torch.logsumexp(x, 1)
            assert ((lse[b, j * G: (j + 1) * G].double() - rl).abs() <= share + 4 * U * rl.abs()).all()
            if weights is not None:
                rw = w_in[b, j, pos].double() + p.sum(0)
                assert ((w_out[b, j, pos].double() - rw).abs() <= share * p.sum(0) + (G + 1) * U * rw).all()
    return out, lse


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D,H,Hkv,page,layout", [
    (64, 12, 12, 16, "heads"), (128, 8, 2, 16, "slots"), (128, 32, 2, 64, "heads"), (256, 3, 1, 24, "slots"),
    (96, 10, 2, 7, "heads"), (8, 20, 1, 1, "heads"), (128, 40, 1, 256, "slots"), (64, 5, 5, 33, "slots")])
def test_attention_matches_definition(gae, dtype, D, H, Hkv, page, layout):
    """Lengths of none, one, the ends of pages and tiles, past the table; weights added to a second buffer."""
    lens = [0, 1, page, page + 1, 63, 64, 65, 500, 1000, 5000, -3]
    M = (700 + page - 1) // page
    g = _gen(D + H + page)
    k, v = _pools(len(lens) * M + 3, Hkv, page, D, dtype, g, layout)
    table = _table(len(lens), M, k.shape[0], g)
    q = torch.randn(len(lens), H, D, device="cuda", generator=g).to(dtype)
    lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    _check_attention(gae, q, k, v, table, lens)
    w = torch.rand(len(lens), Hkv, M * page + 5, device="cuda", generator=g)
    _check_attention(gae, q, k, v, table, lens, weights=w, weights_out=w.clone())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,H,Hkv,D,n", [(1, 4, 1, 128, 30000), (3, 8, 4, 64, 9001), (2, 2, 2, 256, 5000), (150, 4, 2, 64, 130)])
def test_attention_over_long_and_many_sequences(gae, dtype, B, H, Hkv, D, n):
    """Rows split over many blocks, and many short rows to a block; weights in place."""
    g, page = _gen(n), 16
    M = (n + page - 1) // page
    k, v = _pools(B * M + 1, Hkv, page, D, dtype, g)
    table = _table(B, M, B * M + 1, g)
    q = torch.randn(B, H, D, device="cuda", generator=g).to(dtype)
    lens = torch.tensor([max(0, n - 37 * b) for b in range(B)], dtype=torch.int32, device="cuda")
    w = torch.rand(B, Hkv, M * page, device="cuda", generator=g)
    _check_attention(gae, q, k, v, table, lens, weights=w)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("cap", [64, 192, 193, 384, 385])
def test_attention_of_short_rows(gae, dtype, cap):
    """Tables around the longest row that one block takes whole, few rows and more rows than blocks."""
    for B, H, Hkv, D in ((5, 6, 2, 128), (120, 20, 5, 64)):
        g = _gen(cap + B)
        k, v = _pools(B * cap // 8 + 9, Hkv, 8, D, dtype, g)
        M = -(-cap // 8)
        table = _table(B, M, k.shape[0], g) if B * M <= k.shape[0] else \
            torch.randint(0, k.shape[0], (B, M), device="cuda", generator=g, dtype=torch.int32)
        q = torch.randn(B, H, D, device="cuda", generator=g).to(dtype)
        lens = torch.tensor([(b * 67 + 11) % (cap + 2) for b in range(B)], dtype=torch.int32, device="cuda")
        lens[0] = 0
        _check_attention(gae, q, k, v, table, lens)


def test_attention_passes_over_pages_that_hold_nothing(gae):
    g, B, Hkv, page, D = _gen(3), 4, 2, 16, 128
    k, v = _pools(40, Hkv, page, D, torch.bfloat16, g)
    table = _table(B, 9, 40, g)
    table[0, 0], table[0, 3:6], table[1, :], table[2, 8], table[3, 4] = -1, -7, -1, 40, 2 ** 31 - 1
    q = torch.randn(B, 4, D, device="cuda", generator=g).bfloat16()
    lens = torch.tensor([140, 144, 129, 77], dtype=torch.int32, device="cuda")
    _check_attention(gae, q, k, v, table, lens, weights=torch.rand(B, Hkv, 144, device="cuda", generator=g))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("junk", [math.nan, math.inf, -math.inf])
def test_attention_ignores_what_lies_behind_the_length(gae, dtype, junk):
    """The unused slots of the last page, and all other pages, hold NaN or infinities."""
    g, B, Hkv, page, D = _gen(4), 3, 2, 32, 128
    k, v = _pools(30, Hkv, page, D, dtype, g)
    table = _table(B, 4, 30, g)
    lens = torch.tensor([1, 33, 100], dtype=torch.int32, device="cuda")
    used = torch.zeros(30, page, dtype=torch.bool, device="cuda")
    for b, n in enumerate(lens.tolist()):
        pos = torch.arange(n, device="cuda")
        used[table[b].long()[pos // page], pos % page] = True
    for t in (k, v):
        t.masked_fill_(~used[:, None, :, None], junk)
    q = torch.randn(B, 6, D, device="cuda", generator=g).to(dtype)
    _check_attention(gae, q, k, v, table, lens, weights=torch.rand(B, Hkv, 128, device="cuda", generator=g))


def test_attention_spreads_nan_to_its_own_row_alone(gae):
    """A NaN key gives its sequence's head NaN, as the formula does, and no other."""
    g, Hkv, page, D = _gen(5), 2, 16, 64
    k, v = _pools(8, Hkv, page, D, torch.bfloat16, g)
    table = _table(2, 3, 8, g)
    q = torch.randn(2, 4, D, device="cuda", generator=g).bfloat16()
    lens = torch.tensor([40, 40], dtype=torch.int32, device="cuda")
    k[table[0, 1].long(), 1, 3] = math.nan
    out, lse = gae.paged_attention(q, k, v, table, lens, return_lse=True)
    assert out[0, 2:].isnan().all() and lse[0, 2:].isnan().all()
    assert out[0, :2].isfinite().all() and out[1].isfinite().all() and lse[1].isfinite().all()


def test_attention_with_large_and_equal_scores(gae):
    """Scores far apart (one key takes all) and all equal (scale 0: a plain mean)."""
    g, page, D = _gen(6), 16, 128
    k, v = _pools(30, 1, page, D, torch.bfloat16, g)
    table = _table(1, 20, 30, g)
    q = torch.randn(1, 4, D, device="cuda", generator=g).bfloat16()
    lens = torch.tensor([300], dtype=torch.int32, device="cuda")
    _check_attention(gae, q, k, v, table, lens, scale=0.0)
    _check_attention(gae, q, k, v, table, lens, scale=40.0)


def test_attention_strided_views_shared_pages_and_given_outputs(gae):
    """q and out as slices of wider tensors, two sequences on the same pages, a table that is a slice."""
    g, Hkv, page, D = _gen(7), 2, 16, 128
    k, v = _pools(20, Hkv, page, D, torch.float16, g, "slots")
    wide = _table(1, 12, 20, g).expand(3, 12).contiguous()
    table = wide[:, 2:9]
    qkv = torch.randn(3, 8, D, device="cuda", generator=g).half()
    q, buf = qkv[:, 1:5], torch.full((3, 6, D), 7.0, device="cuda", dtype=torch.float16)
    lens = torch.tensor([112, 50, 112], dtype=torch.int32, device="cuda")
    out = buf[:, 1:5]
    lse = torch.empty(3, 4, device="cuda")
    got = gae.paged_attention(q, k, v, table, lens, out=out, lse=lse, return_lse=True)
    assert got[0] is out and got[1] is lse
    _check_attention(gae, q, k, v, table, lens, got=got)
    assert (buf[:, 0] == 7).all() and (buf[:, 5] == 7).all()


def test_attention_rows_past_32_bit_offsets(gae):
    """Pages whose rows lie beyond 2^31 elements (and 2^32 bytes) of the pool."""
    g, page, D = _gen(8), 64, 128
    P = (2 ** 31 + 2 ** 20) // (page * D) + 1
    k = torch.empty(P, 1, page, D, dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    table = torch.tensor([[P - 1, 0, P - 2, 5], [P - 3, P - 4, 7, 9]], dtype=torch.int32, device="cuda")
    for t in (k, v):
        for pg in table.flatten().tolist():
            t[pg] = torch.randn(1, page, D, device="cuda", generator=g).bfloat16()
    lens = torch.tensor([200, 256], dtype=torch.int32, device="cuda")
    q = torch.randn(2, 4, D, device="cuda", generator=g).bfloat16()
    _check_attention(gae, q, k, v, table, lens)
    new = torch.randn(2, 1, 3, D, device="cuda", generator=g).bfloat16()
    gae.paged_append(new, -new, k, v, table, torch.tensor([0, 62], dtype=torch.int32, device="cuda"))
    assert torch.equal(k[P - 1, 0, :3], new[0, 0]) and torch.equal(v[P - 4, 0, 0], -new[1, 0, 2])
    w = torch.rand(2, 1, 256, device="cuda", generator=g)
    dst = torch.tensor([[P - 6], [P - 7]], dtype=torch.int32, device="cuda")
    _, kept, _ = gae.paged_evict(k, v, table, lens, w, dst, keep=20, recent=5)
    pos = kept[0, 0].long()
    assert torch.equal(k[P - 6, 0, :20], k[table[0].long()[pos // page], 0, pos % page])


def test_attention_is_the_same_every_time(gae):
    g, page = _gen(9), 16
    k, v = _pools(700, 2, page, 128, torch.bfloat16, g)
    table = _table(3, 200, 700, g)
    q = torch.randn(3, 8, 128, device="cuda", generator=g).bfloat16()
    lens = torch.tensor([3200, 1501, 17], dtype=torch.int32, device="cuda")
    w = torch.zeros(3, 2, 3200, device="cuda")
    a = gae.paged_attention(q, k, v, table, lens, return_lse=True, weights=w, weights_out=w.clone())
    for _ in range(5):
        b = gae.paged_attention(q, k, v, table, lens, return_lse=True, weights=w, weights_out=w.clone())
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_attention_of_nothing(gae):
    """No sequences, no pages to a sequence, no pages at all."""
    g, D = _gen(10), 64
    k, v = _pools(4, 2, 16, D, torch.bfloat16, g)
    z = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    q = torch.randn(3, 4, D, device="cuda", generator=g).bfloat16()
    assert gae.paged_attention(q[:0], k, v, z(0, 5), z(0)).shape == (0, 4, D)
    for kk, table in ((k, z(3, 0)), (k[:0], z(3, 5))):
        w = torch.rand(3, 2, 80, device="cuda")
        was = w.clone()
        out, lse = gae.paged_attention(q, kk, kk, table, z(3) + 50, return_lse=True, weights=w)
        assert (out == 0).all() and (lse == -math.inf).all() and torch.equal(w, was)
    gae.paged_append(q[:, :2, None], q[:, :2, None], k[:0], v[:0], z(3, 5), z(3))
    new, kept, kw = gae.paged_evict(k[:0], v[:0], z(3, 5), z(3) + 9, torch.rand(3, 2, 80, device="cuda"), z(3, 1), keep=4)
    assert (new == 0).all() and (kept == -1).all() and (kw == 0).all()


def test_strides_of_single_elements_are_not_looked_at(gae):
    g, D = _gen(11), 64
    odd = lambda t, *st: t.as_strided(t.shape, st)  # noqa: E731
    k, v = _pools(1, 1, 32, D, torch.bfloat16, g)
    k, v = odd(k, 7, 3, D, 1), odd(v, 5, 1, D, 1)
    q = odd(torch.randn(1, 1, D, device="cuda", generator=g).bfloat16(), 3, 9, 1)
    table, lens = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.tensor([20], dtype=torch.int32, device="cuda")
    _check_attention(gae, q, k, v, table, lens)
    new = odd(torch.randn(1, 1, 1, D, device="cuda", generator=g).bfloat16(), 1, 3, 5, 1)
    gae.paged_append(new, new, k, v, table, lens)
    assert torch.equal(k[0, 0, 20], new[0, 0, 0])
    qk, kk = odd(q[:, :, None].clone(), 3, 5, 7, 1), odd(k[:, :, :20].clone(), 1, 3, D, 1)
    lse = torch.zeros(1, 1, 1, device="cuda")
    w = gae.attention_key_weights(qk, kk, lse)
    _check_keys(gae, qk, kk, lse, w, False, 0)


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,Hkv,page,T,layout", [(64, 12, 16, 1, "heads"), (128, 2, 7, 45, "slots"), (8, 1, 1, 9, "heads"),
                                                 (256, 3, 64, 130, "slots"), (96, 5, 24, 33, "heads")])
def test_append_writes_its_rows_and_no_others(gae, dtype, D, Hkv, page, T, layout):
    g, B = _gen(D + T), 6
    M = (T + 40) // page + 1
    k, v = _pools(B * M + 4, Hkv, page, D, dtype, g, layout)
    table = _table(B, M, k.shape[0], g)
    table[4, 1:] = -1
    start = torch.tensor([0, 3, page, M * page - 1, 0, -2], dtype=torch.int32, device="cuda")
    counts = torch.tensor([T, T - 1, T, T, T, T + 100], dtype=torch.int32, device="cuda")
    new = torch.randn(B, T, 3, Hkv, D, device="cuda", generator=g).to(dtype)
    kn, vn = new[:, :, 1].transpose(1, 2), new[:, :, 2].transpose(1, 2)
    for c in (counts, None):
        rk, rv = k.clone(), v.clone()
        for b in range(B):
            for t in range(T if c is None else min(T, c[b].item())):
                pos = start[b].item() + t
                if 0 <= pos < M * page and 0 <= table[b, pos // page] < k.shape[0]:
                    pg = table[b, pos // page].item()
                    rk[pg, :, pos % page], rv[pg, :, pos % page] = kn[b, :, t], vn[b, :, t]
        gae.paged_append(kn, vn, k, v, table, start, counts=c)
        assert torch.equal(k, rk) and torch.equal(v, rv)


# ------------------------------------------------------------- key weights
def _check_keys(gae, q, k, lse, w, causal, off, add=None, scale=None):
    """The exponent of a weight is off by at most e of its score, u |lse| from lse itself and 2 u of
    its own size; the sum of n terms by n u."""
    B, H, Nq, D = q.shape
    Hkv, N = k.shape[1], k.shape[2]
    sc = 1 / math.sqrt(D) if scale is None else scale
    for b in range(B):
        for j in range(Hkv):
            ref = torch.zeros(N, dtype=torch.float64, device="cuda")
            tol = torch.zeros_like(ref)
            for h in range(j * (H // Hkv), (j + 1) * (H // Hkv)):
                x = q[b, h].double() @ k[b, j].double().T * sc
                A = q[b, h].double().abs() @ k[b, j].double().abs().T * sc
                l = lse[b, h].double()[:, None]
                p = torch.where(l == -math.inf, 0.0, torch.exp(x - l))
                if causal:
                    rows = torch.arange(Nq, device="cuda")[:, None] + off
                    p = torch.where(torch.arange(N, device="cuda")[None] <= rows, p, 0.0)
                ref += p.sum(0)
                e = (D + 4) * U * A + 4 * U * torch.where(l == -math.inf, 0.0, l.abs()) + 2.0 ** -20
                tol += (p * e).sum(0) + Nq * U * p.sum(0)
            if add is not None:
                ref += add[b, j].double()
            err = (w[b, j].double() - ref).abs()
            assert (err <= tol + 2 * U * ref + 1e-30).all(), (b, j, (err - tol).max().item())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,H,Hkv,Nq,Nkv,D,causal,q_off,kv_off", [
    (2, 3, 3, 256, 256, 128, True, 0, 0), (1, 4, 2, 300, 300, 64, True, 0, 0), (1, 2, 1, 77, 515, 128, True, 438, 0),
    (1, 2, 2, 1, 1, 64, True, 0, 0), (2, 6, 2, 130, 64, 128, False, 0, 0), (1, 2, 1, 1, 1000, 64, True, 999, 0),
    (1, 1, 1, 200, 300, 128, True, 0, 100), (1, 5, 1, 129, 127, 64, False, 0, 0), (1, 2, 2, 700, 40, 128, True, 0, 0),
    (1, 8, 1, 640, 640, 128, True, 0, 0)])
def test_key_weights_match_definition(gae, dtype, B, H, Hkv, Nq, Nkv, D, causal, q_off, kv_off):
    """Odd lengths, grouped heads, offsets: queries before every key, keys behind every query."""
    g = _gen(Nq + Nkv)
    q = torch.randn(B, Nq, H, D, device="cuda", generator=g).to(dtype).transpose(1, 2)
    k = torch.randn(B, Hkv, Nkv, D, device="cuda", generator=g).to(dtype)
    off = q_off - kv_off
    x = q.double() @ k.double().repeat_interleave(H // Hkv, 1).transpose(2, 3) / math.sqrt(D)
    if causal:
        rows = torch.arange(Nq, device="cuda")[:, None] + off
        x = x.masked_fill(torch.arange(Nkv, device="cuda")[None] > rows, -math.inf)
    lse = torch.logsumexp(x, -1).float()
    w = gae.attention_key_weights(q, k, lse, causal=causal, q_offset=q_off, kv_offset=kv_off)
    torch.cuda.synchronize()
    gae.device_status()
    _check_keys(gae, q, k, lse, w, causal, off)
    # added to a slice of a wider buffer, whose other entries stay
    buf = torch.rand(B, Hkv, Nkv + 9, device="cuda", generator=g)
    was = buf.clone()
    r = gae.attention_key_weights(q, k, lse, causal=causal, q_offset=q_off, kv_offset=kv_off, out=buf[:, :, 4: 4 + Nkv],
                                  accumulate=True)
    _check_keys(gae, q, k, lse, r, causal, off, add=was[:, :, 4: 4 + Nkv])
    assert torch.equal(buf[:, :, :4], was[:, :, :4]) and torch.equal(buf[:, :, 4 + Nkv:], was[:, :, 4 + Nkv:])


def test_key_weights_of_the_forwards_lse_sum_to_the_queries(gae):
    """With attention()'s own log-sum-exp every query hands out a weight of one."""
    g, B, H, N, D = _gen(1), 2, 4, 1500, 128
    q, k, v = (torch.randn(B, H, N, D, device="cuda", generator=g).bfloat16() for _ in range(3))
    _, lse = gae.attention(q, k, v, causal=True, return_lse=True)
    w = gae.attention_key_weights(q, k, lse, causal=True)
    # the forward's lse sums 16-bit rounded probabilities: its share is within 2^-8 of one
    assert ((w.sum(-1) / N - 1).abs() <= 2.0 ** -8).all()


def test_key_weights_no_queries_and_infinities(gae):
    g, D = _gen(2), 64
    k = torch.randn(1, 2, 100, D, device="cuda", generator=g).bfloat16()
    empty = torch.empty(1, 2, 0, D, dtype=torch.bfloat16, device="cuda")
    none = torch.empty(1, 2, 0, device="cuda")
    assert (gae.attention_key_weights(empty, k, none) == 0).all()
    buf = torch.full((1, 2, 100), 3.0, device="cuda")
    gae.attention_key_weights(empty, k, none, out=buf, accumulate=True)
    assert (buf == 3).all()
    # rows that saw no key (lse -inf) add nothing; keys behind every query may hold anything
    q = torch.randn(1, 2, 90, D, device="cuda", generator=g).bfloat16()
    k[:, :, 95:] = math.nan
    lse = torch.full((1, 2, 90), 8.0, device="cuda")
    lse[:, :, 10:20] = -math.inf
    w = gae.attention_key_weights(q, k, lse, causal=True, q_offset=4)
    assert (w[:, :, 94:] == 0).all() and w.isfinite().all()
    _check_keys(gae, q, k[:, :, :94], lse, w[:, :, :94], True, 4)
    w = gae.attention_key_weights(q, k, lse, causal=True, kv_offset=1000)  # no query sees any key
    assert (w == 0).all()


# ---------------------------------------------------------------- eviction
def _evict_reference(k, v, table, lens, w, dst, keep, recent):
    B, Hkv, page, P = table.shape[0], k.shape[1], k.shape[2], k.shape[0]
    rk, rv = k.clone(), v.clone()
    new = torch.zeros(B, dtype=torch.int32)
    kept = torch.full((B, Hkv, keep), -1, dtype=torch.int32)
    kw = torch.zeros(B, Hkv, keep)
    tb, db = table.tolist(), dst.tolist()
    for b, n in enumerate(lens.tolist()):
        n = max(0, min(n, table.shape[1] * page, w.shape[2]))
        here = [t for t in range(n) if 0 <= tb[b][t // page] < P]
        new[b] = min(keep, len(here))
        for j in range(Hkv):
            wj = w[b, j, :n].tolist()
            order = sorted(here, key=lambda t: (t < n - recent, not math.isnan(wj[t]),
                                                -wj[t] if not math.isnan(wj[t]) else 0.0, t))
            for i, t in enumerate(sorted(order[:keep])):
                kept[b, j, i], kw[b, j, i] = t, wj[t]
                pg = db[b][i // page]
                if 0 <= pg < P:
                    rk[pg, j, i % page], rv[pg, j, i % page] = k[tb[b][t // page], j, t % page], v[tb[b][t // page], j, t % page]
    return rk, rv, new, kept, kw


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,Hkv,page,n,keep,recent", [
    (64, 3, 16, 300, 100, 10), (128, 2, 7, 500, 499, 499), (8, 1, 1, 90, 1, 0), (256, 1, 24, 300, 300, 0),
    (128, 2, 64, 1030, 1025, 1), (96, 2, 16, 5000, 40, 40), (64, 1, 32, 20000, 9000, 100)])
def test_evict_keeps_the_heaviest(gae, dtype, D, Hkv, page, n, keep, recent):
    """Random, equal, zero of both signs, negative, infinite and NaN weights; lengths around keep."""
    g = _gen(n + keep)
    kinds = ["random", "equal", "few", "odd"]
    B = len(kinds) + 4
    M, Md = (n + page - 1) // page, (keep + page - 1) // page
    k, v = _pools(B * (M + Md) + 2, Hkv, page, D, dtype, g)
    both = _table(B, M + Md, k.shape[0], g)
    table, dst = both[:, :M].contiguous(), both[:, M:]
    w = torch.rand(B, Hkv, n, device="cuda", generator=g) ** 6
    w[1] = 0.25
    w[2] = torch.randint(0, 3, w[2].shape, device="cuda", generator=g).float()
    w[3] -= 0.3
    w[3, :, ::5], w[3, :, 1::7], w[3, :, 2::11], w[3, :, 3::13], w[3, :, 4::17] = 0.0, -0.0, math.nan, math.inf, -math.inf
    lens = torch.tensor([n, n, n, n, 0, 1, keep, min(n, keep + 1)], dtype=torch.int32, device="cuda")
    ref = _evict_reference(k.cpu(), v.cpu(), table.cpu(), lens.cpu(), w.cpu(), dst.cpu(), keep, recent)
    new, kept, kw = gae.paged_evict(k, v, table, lens, w, dst, keep=keep, recent=recent)
    torch.cuda.synchronize()
    gae.device_status()
    assert torch.equal(new.cpu(), ref[2]) and torch.equal(kept.cpu(), ref[3])
    assert torch.equal(kw.cpu().nan_to_num(nan=5.0), ref[4].nan_to_num(nan=5.0))
    assert torch.equal(k.cpu(), ref[0]) and torch.equal(v.cpu(), ref[1])


def test_evict_passes_over_pages_that_hold_nothing(gae):
    g, page, D, n, keep = _gen(12), 16, 64, 160, 70
    k, v = _pools(60, 2, page, D, torch.bfloat16, g)
    both = _table(3, 15, 60, g)
    table, dst = both[:, :10].contiguous(), both[:, 10:].contiguous()
    table[0, 2:5], table[1, :], table[2, 1:9] = -1, 60, -5
    dst[2, 1] = -1  # a destination that names no page drops its rows
    w = torch.rand(3, 2, n, device="cuda", generator=g)
    lens = torch.tensor([n, n, n - 3], dtype=torch.int32, device="cuda")
    ref = _evict_reference(k.cpu(), v.cpu(), table.cpu(), lens.cpu(), w.cpu(), dst.cpu(), keep, 20)
    new, kept, kw = gae.paged_evict(k, v, table, lens, w, dst, keep=keep, recent=20)
    assert torch.equal(new.cpu(), ref[2]) and torch.equal(kept.cpu(), ref[3]) and torch.equal(kw.cpu(), ref[4])
    assert torch.equal(k.cpu(), ref[0]) and torch.equal(v.cpu(), ref[1])


def test_evict_of_very_long_sequences(gae):
    """More keys than one block's shared memory holds, few and many of them kept."""
    g, page, D, n = _gen(13), 64, 8, 400_000
    M = (n + page - 1) // page
    k, v = _pools(2 * M + 2000, 1, page, D, torch.bfloat16, g)
    both = _table(1, M + 1500, k.shape[0], g)
    w = torch.rand(1, 1, n, device="cuda", generator=g) ** 4
    w[0, 0, ::3] = 0.5
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    for keep, recent in ((70_000, 64), (150, 0)):
        new, kept, kw = gae.paged_evict(k, v, both[:, :M].contiguous(), lens, w, both[:, M:], keep=keep, recent=recent)
        x = w[0, 0].clone()
        x[n - recent:] = math.inf
        want = torch.sort(x, descending=True, stable=True).indices[:keep].sort().values
        assert new.item() == keep and torch.equal(kept[0, 0].long(), want) and torch.equal(kw[0, 0], w[0, 0][want])
        at = torch.arange(keep, device="cuda")
        dk = k[both[0, M:].long()[at // page], 0, at % page]
        assert torch.equal(dk, k[both[0].long()[want // page], 0, want % page])


# --------------------------------------------------------- streams, graphs
def test_on_another_stream_and_captured(gae):
    """Every operator on a side stream, two decoding steps at once, and a captured run replayed
    after its lengths and inputs changed in place."""
    g, B, Hkv, page, D, M = _gen(20), 3, 2, 16, 128, 40
    k, v = _pools(B * M + 60, Hkv, page, D, torch.bfloat16, g)
    both = _table(B, M + 8, k.shape[0], g)
    table, dst = both[:, :M].contiguous(), both[:, M:].contiguous()
    q = torch.randn(B, 8, D, device="cuda", generator=g).bfloat16()
    lens = torch.tensor([600, 17, 333], dtype=torch.int32, device="cuda")
    w = torch.rand(B, Hkv, M * page, device="cuda", generator=g)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    r1 = gae.paged_attention(q, k, v, table, lens, return_lse=True, stream=s1)
    r2 = gae.paged_attention(q.flip(0).contiguous(), k, v, table, lens, return_lse=True, stream=s2)
    torch.cuda.synchronize()
    _check_attention(gae, q, k, v, table, lens, got=r1)
    _check_attention(gae, q.flip(0), k, v, table, lens, got=r2)

    # append, key weights and eviction on a stream of their own, the weights a slice of a wider buffer
    rows = torch.randn(B, Hkv, 5, D, device="cuda", generator=g).bfloat16()
    wide = torch.rand(B, Hkv, M * page + 3, device="cuda", generator=g)
    part = wide[:, :, 3:]
    lse = torch.full((B, 8, 70), 6.0, device="cuda")
    qq, kk = (torch.randn(B, h, n, D, device="cuda", generator=g).bfloat16() for h, n in ((8, 70), (Hkv, 90)))
    torch.cuda.synchronize()
    gae.paged_append(rows, -rows, k, v, table, lens, stream=s1)
    was = part.clone()
    s1.synchronize()
    o2 = gae.paged_attention(q, k, v, table, lens + 5, return_lse=True, weights=part, stream=s1)
    kw2 = gae.attention_key_weights(qq, kk, lse, causal=True, q_offset=20, stream=s1)
    s1.synchronize()
    ref = _evict_reference(k.cpu(), v.cpu(), table.cpu(), lens.cpu(), part.cpu(), dst.cpu(), 90, 3)
    e2 = gae.paged_evict(k, v, table, lens, part, dst, keep=90, recent=3, stream=s1)
    torch.cuda.synchronize()
    for b, n in enumerate(lens.tolist()):
        assert torch.equal(k[table[b, (n + 4) // page].long(), :, (n + 4) % page], rows[b, :, 4])
    _check_attention(gae, q, k, v, table, lens + 5, got=o2)
    assert ((part - was).sum(-1) - 4).abs().max() <= 1e-3  # four query heads' weights of one each
    _check_keys(gae, qq, kk, lse, kw2, True, 20)
    assert torch.equal(e2[1].cpu(), ref[3]) and torch.equal(k.cpu(), ref[0]) and torch.equal(v.cpu(), ref[1])

    new = torch.randn(B, Hkv, 1, D, device="cuda", generator=g).bfloat16()
    after = lens + 1
    w2 = w.clone()

    def step():
        gae.paged_append(new, -new, k, v, table, lens)
        o, lse = gae.paged_attention(q, k, v, table, after, return_lse=True, weights=w, weights_out=w2)
        return o, lse, gae.paged_evict(k, v, table, after, w2, dst, keep=100, recent=8)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, lse, (n2, kept, kw) = step()
    for turn in range(2):
        lens.copy_(torch.tensor([[500, 0, 200], [639, 64, 15]][turn], dtype=torch.int32))
        after.copy_(lens + 1)
        q.copy_(torch.randn(B, 8, D, device="cuda", generator=g))
        new.copy_(torch.randn(B, Hkv, 1, D, device="cuda", generator=g))
        w2.copy_(w)
        graph.replay()
        torch.cuda.synchronize()
        for b, n in enumerate(lens.tolist()):
            assert torch.equal(k[table[b, n // page].long(), :, n % page], new[b, :, 0])
        _check_attention(gae, q, k, v, table, after, got=(o, lse))
        ref = _evict_reference(k.cpu(), v.cpu(), table.cpu(), after.cpu(), w2.cpu(), dst.cpu(), 100, 8)
        assert torch.equal(n2.cpu(), ref[2]) and torch.equal(kept.cpu(), ref[3])
        assert torch.equal(k.cpu(), ref[0]) and torch.equal(v.cpu(), ref[1])


# ------------------------------------------------------ a run of them together
def _layers(gae, n, D, H, F):
    """Weights larger than the usual 0.02, so that attention and its scores matter."""
    layers = [gae.Gpt2Layer.random(D, H, F, seed=50 + i) for i in range(n)]
    for layer in layers:
        layer.w["w_qkv"].mul_(4)
    return layers


@pytest.mark.parametrize("D,H,page", [(256, 4, 16), (512, 4, 24)])
def test_stack_decodes_what_it_computes_whole(gae, D, H, page):
    """A prompt of ragged lengths, then token by token, against the stack over the whole sequence
    (the layer tolerance of tests/test_layer_gpu.py: 2e-2 * max(1, |ref|))."""
    B, S, steps, g = 3, 150, 9, _gen(30)
    layers = _layers(gae, 2, D, H, 1024)
    counts = [150, 33, 1]
    x = torch.randn(B, S + steps, D, device="cuda", generator=g).bfloat16()
    cache = gae.PagedKVCache(2, B, H, D // H, S + steps, page_size=page)
    whole = [gae.layer_stack_forward(layers, x[b: b + 1, : counts[b] + steps].contiguous())[0].float() for b in range(B)]
    close = lambda a, r: ((a.float() - r).abs() <= 2e-2 * r.abs().clamp(min=1)).all()  # noqa: E731
    prompt = torch.zeros(B, S, D, device="cuda", dtype=torch.bfloat16)
    for b, n in enumerate(counts):
        prompt[b, :n] = x[b, :n]
    y = gae.layer_stack_prefill(layers, prompt, cache, counts)
    for b, n in enumerate(counts):
        assert close(y[b, :n], whole[b][:n]), b
    for t in range(steps):
        y = gae.layer_stack_decode(layers, torch.stack([x[b, n + t] for b, n in enumerate(counts)]), cache)
        for b, n in enumerate(counts):
            assert close(y[b], whole[b][n + t]), (t, b)
    torch.cuda.synchronize()
    gae.device_status()
    assert cache.lens.tolist() == cache.lengths == [n + steps for n in counts]
    with pytest.raises(gae.GAEError):
        gae.layer_stack_decode(layers, x[:, 0].contiguous(), cache)  # no room left


def _dense(cache, layer):
    """(key, value) lists per sequence in 64 bits, read through the cache's table."""
    return [tuple(t.double().transpose(0, 1) for t in _rows(cache.k[layer], cache.v[layer], cache.table, b, n)[1:])
            for b, n in enumerate(cache.lens.tolist())]


def test_cache_within_a_budget(gae):
    """Prompt, eviction, decoding past the budget and eviction again: the kept rows are those of the
    heaviest keys, the weights are theirs, and decoding attends to exactly them."""
    B, H, D, S, budget, recent, g = 2, 4, 256, 200, 64, 8, _gen(31)
    layers = _layers(gae, 2, D, H, 512)
    cache = gae.PagedKVCache(2, B, H, D // H, 256, page_size=16, budget=budget, recent=recent)
    counts = [200, 90]
    gae.layer_stack_prefill(layers, torch.randn(B, S, D, device="cuda", generator=g).bfloat16(), cache, counts)
    for w in cache.weights:  # every real query hands out a weight of one per head (lse of 16-bit probabilities)
        assert ((w.sum(-1) / torch.tensor(counts, device="cuda")[:, None] - 1).abs() <= 2.0 ** -7).all()
        assert (w[1, :, 90:] == 0).all()
    for turn in range(2):
        before = [(_dense(cache, i), cache.weights[i].clone()) for i in range(2)]
        was = list(cache.lengths)
        kept = cache.evict()
        assert cache.lengths == [min(n, budget) for n in was] == cache.lens.tolist()
        for i in range(2):
            rows, w = before[i]
            after = _dense(cache, i)
            for b, n in enumerate(was):
                m = min(n, budget)
                for h in range(H):
                    x = w[b, h, :n].clone()
                    x[n - recent:] = math.inf
                    want = torch.sort(x, descending=True, stable=True).indices[:m].sort().values
                    assert torch.equal(kept[i][b, h, :m].long(), want)
                    assert torch.equal(after[b][0][h], rows[b][0][h][want])
                    assert torch.equal(after[b][1][h], rows[b][1][h][want])
                    assert torch.equal(cache.weights[i][b, h, :m], w[b, h, want])
        for _ in range(10):
            gae.layer_stack_decode(layers, torch.randn(B, D, device="cuda", generator=g).bfloat16(), cache)
        assert cache.lengths == [budget + 10] * B
        # one more token by hand: attention over what the cache now holds
        q = torch.randn(B, H, D // H, device="cuda", generator=g).bfloat16()
        w = cache.weights[1].clone()
        cache.next_lens.copy_(cache.lens)
        out = cache.attend(1, q)
        for b in range(B):
            k, v = _dense(cache, 1)[b]
            p = torch.softmax(torch.einsum("hd,hnd->hn", q[b].double(), k) / math.sqrt(D // H), -1)
            assert ((out[b].double() - torch.einsum("hn,hnd->hd", p, v)).abs() <= 2.0 ** -8 * v.abs().max()).all()
            assert ((cache.weights[1][b, :, : budget + 10] - w[b, :, : budget + 10] - p).abs() <= 1e-4).all()


def test_decoding_step_in_a_graph(gae):
    """A captured decoding step replayed token by token gives what the eager steps give."""
    B, H, D, steps, g = 2, 4, 256, 20, _gen(32)
    layers = _layers(gae, 2, D, H, 512)
    x = torch.randn(steps, B, D, device="cuda", generator=g).bfloat16()
    eager, graphed = (gae.PagedKVCache(2, B, H, D // H, 64, budget=64) for _ in range(2))
    want = [gae.layer_stack_decode(layers, x[t], eager) for t in range(steps)]
    xin = x[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        gae.layer_stack_decode(layers, xin, graphed)  # token 0, and the warm-up
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = gae.layer_stack_decode(layers, xin, graphed)
    for t in range(1, steps):
        xin.copy_(x[t])
        graph.replay()
        assert torch.equal(y, want[t]), t
    for a, b in zip(eager.weights, graphed.weights):
        assert torch.equal(a, b)
    assert graphed.lengths != [steps] * B  # the host has not seen the replays
    graphed.refresh()
    assert graphed.lengths == graphed.lens.tolist() == [steps] * B


# What key weights are made of, in tiles of 128 queries that every key sees and in the others: 384 queries, of which
# the third tile is cut by the mask, against 256 keys (causal: query row r sees key c iff c <= r + 128).
def _full_tiles(seed, dtype=torch.bfloat16, D=64):
    g = _gen(seed)
    q = torch.randn(1, 2, 384, D, device="cuda", generator=g).to(dtype)
    k = torch.randn(1, 1, 256, D, device="cuda", generator=g).to(dtype)
    return q, k, torch.full((1, 2, 384), 6.0, device="cuda")


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_key_weights_of_queries_that_saw_nothing_are_nothing(gae, dtype, causal):
    """A query whose lse is -inf adds exactly nothing, whatever it holds and wherever it stands: the
    other queries' weights are the same bits, keys that only such queries see have a weight of 0."""
    q, k, lse = _full_tiles(40, dtype)
    kw = dict(causal=causal, q_offset=128 if causal else 0)
    assert (gae.attention_key_weights(q, k, torch.full_like(lse, -math.inf), **kw) == 0).all()
    out = torch.arange(lse.shape[2], device="cuda") % 7 == 3  # rows of every tile, and all of the last one
    out[256:] = True
    lse[:, :, out] = -math.inf
    want = gae.attention_key_weights(q, k, lse, **kw)
    _check_keys(gae, q, k, lse, want, causal, kw["q_offset"])
    for junk in (math.nan, math.inf, -math.inf, 0.0):
        q2 = q.clone()
        q2[:, :, out] = junk
        assert torch.equal(gae.attention_key_weights(q2, k, lse, **kw), want), junk


def test_key_weights_of_a_nan_query_are_nan_at_every_column(gae):
    """A NaN query (its lse is NaN too) makes every key that sees it NaN, in whole tiles and cut ones alike."""
    q, k, lse = _full_tiles(41)
    for row in range(256):
        q2, l2 = q.clone(), lse.clone()
        q2[0, 1, row], l2[0, 1, row] = math.nan, math.nan
        w = gae.attention_key_weights(q2, k, l2)
        assert w.isnan().all(), row
        w = gae.attention_key_weights(q2, k, l2, causal=True, q_offset=128)
        seen = torch.arange(256, device="cuda") <= row + 128
        assert w[0, 0, seen].isnan().all() and w[0, 0, ~seen].isfinite().all(), row
        w = gae.attention_key_weights(q2, k, lse)  # a NaN query whose lse is finite
        assert w.isnan().all(), row


@pytest.mark.parametrize("row", [0, 1, 2, 3, 4, 5, 30, 31, 100, 127, 128, 300, 383])
def test_key_weights_of_scores_far_above_the_lse(gae, row):
    """An lse that does not cover the keys (a part's, before a merge): weights as large as fp32 has them,
    then +inf, from any column.  fp32 ends at e^88.72."""
    q, k, lse = _full_tiles(42)
    q.zero_()  # every score is 0: a weight is exp(-lse)
    for l, want in ((-87.0, math.exp(87.0)), (-88.5, math.exp(88.5)), (-89.0, math.inf), (-97.0, math.inf),
                    (-150.0, math.inf), (-3e38, math.inf)):
        l2 = lse.clone()
        l2[0, 0, row] = l
        w = gae.attention_key_weights(q, k, l2).double()
        # the exponent's argument is off by 4 u |lse| at most, the exponential by 2^-20
        assert (w == want).all() if want == math.inf else ((w / want - 1).abs() <= 4 * U * 90 + 2.0 ** -20).all(), l
    l2 = lse.clone()
    l2[0, 0, row] = math.inf  # a row that saw an infinite score: exp(-inf)
    others = torch.ones(384, dtype=torch.bool, device="cuda")
    others[row] = False
    want = 2 * 384 * math.exp(-6.0) - math.exp(-6.0)
    w = gae.attention_key_weights(q, k, l2).double()
    assert ((w / want - 1).abs() <= 4 * U * 6 + 2.0 ** -20 + 768 * U).all()


def test_key_weights_of_far_scores_are_nothing(gae):
    """Weights below fp32's smallest normal number come out as 0, from any column."""
    q, k, lse = _full_tiles(43)
    q.zero_()
    lse.fill_(104.0)
    assert (gae.attention_key_weights(q, k, lse) == 0).all()


def test_evict_from_host_threads(gae):
    """Caches of very different lengths evicted at the same time through the C entry, by a thread and on a
    stream each: no call may lose its launch to another's."""
    g, page, D, turns = _gen(45), 16, 64, 3000
    cases = []
    for n, keep in ((500, 20), (39_000, 20)) * 3:
        M = (n + page - 1) // page
        k, v = _pools(M + 2, 1, page, D, torch.bfloat16, g)
        both = _table(1, M + 2, M + 2, g)
        w = torch.rand(1, 1, n, device="cuda", generator=g)
        lens = torch.tensor([n], dtype=torch.int32, device="cuda")
        new, kept = torch.zeros_like(lens), torch.zeros(1, 1, keep, dtype=torch.int32, device="cuda")
        kw = torch.zeros(1, 1, keep, device="cuda")
        pool = gae.KvPool(k.data_ptr(), v.data_ptr(), tuple(k.stride()[:3]), tuple(v.stride()[:3]), *k.shape, gae.DTYPE_BF16)
        args = gae.PagedEvictArgs(1, both.data_ptr(), M + 2, M, lens.data_ptr(), w.data_ptr(), (n, n), n,
                                  both.data_ptr() + 4 * M, M + 2, 2, keep, 0, new.data_ptr(), kept.data_ptr(), kw.data_ptr())
        want = torch.sort(w[0, 0], descending=True, stable=True).indices[:keep].sort().values
        cases.append((pool, args, torch.cuda.Stream(), kept, want, (k, v, both, w, lens, new, kw)))
    torch.cuda.synchronize()
    L, status = gae.lib(), []

    def work(pool, args, stream):
        st = stream.cuda_stream
        status.extend({L.gae_paged_evict(ctypes.byref(pool), ctypes.byref(args), st) for _ in range(turns)})

    threads = [threading.Thread(target=work, args=c[:3]) for c in cases]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert status == [0] * len(cases)
    for c in cases:
        assert torch.equal(c[3][0, 0].long(), c[4])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("below", [14, 20, 24, 28])
def test_attention_of_many_light_keys_beside_heavy_ones(gae, dtype, below):
    """Four keys of the first 64 take nearly all of each probability and their value is 0: the output is the
    sum of very many small probabilities, 2^-below of a heavy key's each.  No term is negative, so the
    file's share holds of the output itself; a f16 probability is besides off by 2^-38 of the heaviest at
    most.  So many rows (of the same pages) that a block has whole ones."""
    B, n, D, page = 888, 131072, 64, 64
    g = _gen(44 + below)
    k, v = _pools(n // page, 1, page, D, dtype, g)
    k.zero_()
    v.abs_()
    table = _table(1, n // page, n // page, g)
    at = table[0, 0].long()
    k[at, 0, 5::16, 0], v[at, 0, 5::16] = 1.0, 0.0
    q = torch.zeros(1, 2, D, device="cuda", dtype=dtype)
    q[0, :, 0] = below + torch.tensor([0.5, 0.25], device="cuda")
    lens = torch.full((B,), n, dtype=torch.int32, device="cuda")
    out = gae.paged_attention(q.expand(B, 2, D), k, v, table.expand(B, -1), lens, scale=math.log(2.0)).double()
    _, kb, vb = _rows(k, v, table, 0, n)
    ref = torch.softmax(q[0].double() @ kb[:, 0].T * math.log(2.0), 1) @ vb[:, 0]
    share = 2 * (D + 4) * U * (below + 1) + (n + 8) * U + 2.0 ** -20 + (2.0 ** -17 if dtype != torch.float32 else 0)
    step = n * 2.0 ** -38 * vb.max() if dtype == torch.float16 else 0.0
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0  # half the output's smallest step
    err = (out - ref).abs()
    assert (err <= (share + torch.finfo(dtype).eps / 2) * ref + step + tiny).all(), (err / ref).max().item()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_weights_are_the_same_every_time(gae, dtype):
    """The weights that attention adds up, and those of a prompt, bit by bit, over split rows and short ones."""
    g, page, B = _gen(46), 16, 3
    k, v = _pools(700, 2, page, 128, dtype, g)
    table = _table(B, 200, 700, g)
    q = torch.randn(B, 8, 128, device="cuda", generator=g).to(dtype)
    lens = torch.tensor([3200, 1501, 17], dtype=torch.int32, device="cuda")
    w = torch.rand(B, 2, 3200, device="cuda", generator=g)
    runs = []
    for _ in range(6):
        out = w.clone()
        gae.paged_attention(q, k, v, table, lens, weights=w, weights_out=out)
        runs.append(out)
    assert not torch.equal(runs[0], w) and all(torch.equal(runs[0], r) for r in runs[1:])
    if dtype == torch.float32:
        return
    qs, ks = (torch.randn(1, h, 900, 128, device="cuda", generator=g).to(dtype) for h in (4, 2))
    lse = torch.full((1, 4, 900), 7.0, device="cuda")
    runs = [gae.attention_key_weights(qs, ks, lse, causal=True) for _ in range(6)]
    assert all(torch.equal(runs[0], r) for r in runs[1:])


def test_a_prompt_padded_past_the_cache(gae):
    """Right padding may be longer than the cache: its rows have no place, and no weight."""
    B, H, D, g = 2, 4, 256, _gen(47)
    layers = _layers(gae, 1, D, H, 512)
    x = torch.randn(B, 80, D, device="cuda", generator=g).bfloat16()
    counts, caches = [60, 33], []
    for S, max_len in ((80, 60), (60, 60)):  # 64 positions of pages; the same prompt with and without the long padding
        cache = gae.PagedKVCache(1, B, H, D // H, max_len, budget=40, recent=4)
        y = gae.layer_stack_prefill(layers, x[:, :S].contiguous(), cache, counts)
        caches.append((cache, y))
    (a, ya), (b, yb) = caches
    assert a.lengths == b.lengths == counts
    for i, n in enumerate(counts):
        assert torch.equal(ya[i, :n], yb[i, :n])
        assert torch.equal(a.weights[0][i, :, :n], b.weights[0][i, :, :n]) and (a.weights[0][i, :, n:] == 0).all()


def test_attend_after_an_eviction(gae):
    """Between steps attend() sees what the cache holds, also right after an eviction."""
    B, H, D, S, budget, g = 2, 4, 256, 100, 32, _gen(48)
    layers = _layers(gae, 1, D, H, 512)
    cache = gae.PagedKVCache(1, B, H, D // H, 128, budget=budget, recent=8)
    gae.layer_stack_prefill(layers, torch.randn(B, S, D, device="cuda", generator=g).bfloat16(), cache)
    cache.evict()
    q = torch.randn(B, H, D // H, device="cuda", generator=g).bfloat16()
    w = cache.weights[0].clone()
    out = cache.attend(0, q)
    for b, (k, v) in enumerate(_dense(cache, 0)):
        p = torch.softmax(torch.einsum("hd,hnd->hn", q[b].double(), k) / math.sqrt(D // H), -1)
        assert ((out[b].double() - torch.einsum("hn,hnd->hd", p, v)).abs() <= 2.0 ** -8 * v.abs().max()).all()
    assert torch.equal(cache.weights[0][:, :, budget:], w[:, :, budget:])


def test_a_sequence_without_a_new_token_draws_no_weights(gae):
    """In a step that only some sequences take part in, the others' row of q is padding: what it holds
    reaches neither their keys' weights nor anyone else's output."""
    B, H, Hkv, D, g = 3, 4, 2, 64, _gen(49)
    cache = gae.PagedKVCache(1, B, Hkv, D, 64, budget=64)
    rows = torch.randn(B, Hkv, 40, D, device="cuda", generator=g).bfloat16()
    cache.reserve(40, [40, 17, 5])
    cache.append(0, rows, rows)
    cache.commit()
    cache.weights[0].copy_(torch.rand(cache.weights[0].shape, device="cuda", generator=g))
    was = cache.weights[0].clone()
    q = torch.randn(B, H, D, device="cuda", generator=g).bfloat16()
    q[1] = math.nan
    cache.reserve(1, [1, 0, 1])
    cache.append(0, rows[:, :, :1], rows[:, :, :1])
    out = cache.attend(0, q)
    cache.commit()
    assert cache.lens.tolist() == cache.lengths == [41, 17, 6]
    assert torch.equal(cache.weights[0][1], was[1])
    assert out[0].isfinite().all() and out[2].isfinite().all()
    for b, n in ((0, 41), (2, 6)):
        drawn = (cache.weights[0][b] - was[b]).double()
        assert ((drawn.sum(-1) - H // Hkv).abs() <= 1e-4).all() and (drawn[:, n:] == 0).all()


def test_a_ragged_step_in_a_graph(gae):
    """reserve(counts) may be captured: a step that only some sequences take part in, replayed."""
    B, H, D, g = 3, 2, 64, _gen(50)
    rows = torch.randn(B, H, 2, D, device="cuda", generator=g).bfloat16()
    q = torch.randn(B, H, D, device="cuda", generator=g).bfloat16()
    eager, graphed = (gae.PagedKVCache(1, B, H, D, 64, budget=64) for _ in range(2))

    def step(cache):
        cache.reserve(2, [2, 0, 1])
        cache.append(0, rows, rows)
        out = cache.attend(0, q)
        cache.commit()
        return out

    want = [step(eager) for _ in range(5)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(graphed)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(graphed)
    for t in range(1, 5):
        graph.replay()
        assert torch.equal(out, want[t]), t
    graphed.refresh()
    assert graphed.lengths == eager.lengths == [10, 0, 5]
    assert torch.equal(eager.weights[0], graphed.weights[0])


def test_broadcast_operands(gae):
    """Strides of 0: one q for all sequences, one lse row for all heads, one prompt for all of the batch."""
    g, B, Hkv, page, D = _gen(51), 3, 2, 16, 64
    k, v = _pools(40, Hkv, page, D, torch.bfloat16, g)
    table = _table(1, 12, 40, g).expand(B, 12)
    q = torch.randn(1, 1, D, device="cuda", generator=g).bfloat16().expand(B, 6, D)
    lens = torch.tensor([1, 100, 192], dtype=torch.int32, device="cuda")
    _check_attention(gae, q, k, v, table, lens)
    qk = torch.randn(1, 1, 200, D, device="cuda", generator=g).bfloat16().expand(2, 4, 200, D)
    kk = torch.randn(1, 1, 300, D, device="cuda", generator=g).bfloat16().expand(2, 2, 300, D)
    lse = torch.full((1, 1, 200), 6.0, device="cuda").expand(2, 4, 200)
    w = gae.attention_key_weights(qk, kk, lse, causal=True, q_offset=100)
    _check_keys(gae, qk, kk, lse, w, True, 100)
    rows = torch.randn(1, 1, 1, D, device="cuda", generator=g).bfloat16().expand(B, Hkv, 3, D)
    own = _table(B, 12, 40, g)
    start = torch.tensor([0, 15, 189], dtype=torch.int32, device="cuda")
    gae.paged_append(rows, rows, k, v, own, start)
    for b, s in enumerate(start.tolist()):
        for t in range(s, s + 3):
            assert torch.equal(k[own[b, t // page].long(), :, t % page], rows[0, :, 0])


def test_two_graphs_of_one_model_at_once(gae):
    """Two captured runs of the same sizes, replayed together on two streams: each has its own workspace."""
    g, Hkv, page, D, M = _gen(52), 2, 16, 128, 100
    runs = []
    for i in range(2):
        k, v = _pools(2 * M, Hkv, page, D, torch.bfloat16, g)
        table = _table(2, M, 2 * M, g)
        q = torch.randn(2, 8, D, device="cuda", generator=g).bfloat16()
        lens = torch.tensor([1600, 900 + i], dtype=torch.int32, device="cuda")
        w = torch.rand(2, Hkv, M * page, device="cuda", generator=g)
        qk, kk = (torch.randn(1, h, 1000, D, device="cuda", generator=g).bfloat16() for h in (4, 2))
        lse = torch.full((1, 4, 1000), 7.0, device="cuda")
        graph, stream, wo = torch.cuda.CUDAGraph(), torch.cuda.Stream(), w.clone()
        call = lambda: (*gae.paged_attention(q, k, v, table, lens, return_lse=True, weights=w, weights_out=wo),  # noqa: B023,E731
                        gae.attention_key_weights(qk, kk, lse, causal=True))  # noqa: B023
        want = [t.clone() for t in (*call(), wo)]
        _check_attention(gae, q, k, v, table, lens, got=want[:2])
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            got = (*call(), wo)
        runs.append((graph, stream, got, want, (k, v, table, q, lens, w, qk, kk, lse)))  # what the graph reads lives on
    for _ in range(20):
        for graph, stream, got, _, kept in runs:
            with torch.cuda.stream(stream):
                for t in got[:3]:
                    t.fill_(-1)
                got[3].copy_(kept[5])  # entries behind a sequence's length are not written
                graph.replay()
    torch.cuda.synchronize()
    for _, _, got, want, _ in runs:
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_decode_and_prefill_of_slices(gae):
    """The last hidden states of a prompt, and every second token of a longer one, taken as they lie."""
    B, H, D, S, g = 3, 4, 256, 20, _gen(53)
    layers = _layers(gae, 2, D, H, 512)
    x = torch.randn(B, 2 * S, D, device="cuda", generator=g).bfloat16()
    got = []
    for take in (lambda t: t, lambda t: t.contiguous()):
        cache = gae.PagedKVCache(2, B, H, D // H, 64, budget=64)
        y = gae.layer_stack_prefill(layers, take(x[:, ::2]), cache)
        got.append((y, gae.layer_stack_decode(layers, take(y[:, -1]), cache), *cache.weights))
    assert all(torch.equal(a, b) for a, b in zip(*got))
