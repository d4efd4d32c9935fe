"""The paged key-value cache's refusals and ctypes mirrors, without a GPU: every
call here is answered by the argument checks before anything is launched."""
import ctypes as C
import os
import subprocess

import pytest

torch = pytest.importorskip("torch")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PTR = 1 << 20  # a 16-byte aligned address that no refused call reads
INVALID, UNSUPPORTED = 1, 2

STRUCTS = [("gae_kv_pool", "KvPool"), ("gae_paged_append_args", "PagedAppendArgs"),
           ("gae_paged_attn_args", "PagedAttnArgs"), ("gae_key_weights_args", "KeyWeightsArgs"),
           ("gae_paged_evict_args", "PagedEvictArgs")]


def test_mirrors_match_the_header(gae, tmp_path):
    lines = ['#include <stddef.h>', '#include <stdio.h>', '#include "gae.h"', "int main(void) {"]
    for cname, pyname in STRUCTS:
        lines.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        for field, _ in getattr(gae, pyname)._fields_:
            lines.append(f'printf("{cname} {field} %zu\\n", offsetof({cname}, {field}));')
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = {}
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines():
        cname, key, val = line.split()
        got[(cname, key)] = int(val)
    for cname, pyname in STRUCTS:
        cls = getattr(gae, pyname)
        assert C.sizeof(cls) == got[(cname, "size")], cname
        for field, _ in cls._fields_:
            assert getattr(cls, field).offset == got[(cname, field)], (cname, field)


def _pool(gae, **kw):
    s = gae.KvPool(PTR, PTR, (C.c_int64 * 3)(2 * 16 * 64, 16 * 64, 64), (C.c_int64 * 3)(2 * 16 * 64, 16 * 64, 64), 10, 2,
                   16, 64, gae.DTYPE_BF16)
    for k, v in kw.items():
        if isinstance(v, tuple):
            getattr(s, k)[:] = v
        else:
            setattr(s, k, v)
    return s


def _args(cls, base, **kw):
    s = cls()
    for k, v in {**base, **kw}.items():
        if isinstance(v, tuple):
            getattr(s, k)[:] = v
        else:
            setattr(s, k, v)
    return s


APPEND = dict(k_new=PTR, v_new=PTR, k_new_stride=(128, 64, 128), v_new_stride=(128, 64, 128), batch=1, tokens=1,
              page_table=PTR, table_stride=4, max_pages=4, start=PTR)
ATTN = dict(q=PTR, o=PTR, q_stride=(256, 64), o_stride=(256, 64), batch=1, heads=4, page_table=PTR, table_stride=4,
            max_pages=4, seq_lens=PTR, scale=0.125, workspace=PTR, workspace_bytes=1 << 30)
KEYS = dict(q=PTR, k=PTR, lse=PTR, out=PTR, batch=1, heads=4, kv_heads=2, seq_q=16, seq_kv=16, head_dim=64,
            q_stride=(4096, 1024, 64), k_stride=(4096, 1024, 64), lse_stride=(64, 16), out_stride=(32, 16), dtype=1,
            scale=0.125, workspace=PTR, workspace_bytes=1 << 30)
EVICT = dict(batch=1, page_table=PTR, table_stride=4, max_pages=4, seq_lens=PTR, weights=PTR, w_stride=(128, 64),
             weights_len=64, dst_table=PTR + 4096, dst_stride=2, dst_max_pages=2, keep=32, recent=4, new_lens=PTR + 64,
             kept=PTR, kept_weights=PTR + 64)

POOL_BAD = [(dict(num_pages=-1), INVALID), (dict(kv_heads=0), INVALID), (dict(page_size=0), INVALID),
            (dict(head_dim=0), INVALID), (dict(head_dim=60), UNSUPPORTED), (dict(head_dim=264), UNSUPPORTED),
            (dict(k=None), INVALID), (dict(v=PTR + 8), INVALID), (dict(k_stride=(2048, 1024, 60)), INVALID),
            (dict(v_stride=(-2048, 1024, 64)), INVALID), (dict(dtype=7), INVALID),
            (dict(num_pages=1 << 31), UNSUPPORTED), (dict(kv_heads=65536), UNSUPPORTED)]


@pytest.mark.parametrize("bad,status", POOL_BAD)
def test_pool_refusals(gae, bad, status):
    L, pool = gae.lib(), _pool(gae, **bad)
    for fn, cls, base in (("gae_paged_append", gae.PagedAppendArgs, APPEND),
                          ("gae_paged_attn_fwd", gae.PagedAttnArgs, ATTN),
                          ("gae_paged_evict", gae.PagedEvictArgs, EVICT)):
        a = _args(cls, base, **({"heads": 65536 * 4} if "kv_heads" in bad and fn == "gae_paged_attn_fwd" else {}))
        assert getattr(L, fn)(C.byref(pool), C.byref(a), None) == status, fn


def _refused(gae, fn, cls, base, bad, status):
    a = _args(cls, base, **bad)
    assert getattr(gae.lib(), fn)(C.byref(_pool(gae)), C.byref(a), None) == status
    assert gae.lib().gae_last_error(None, 0) == status


@pytest.mark.parametrize("bad,status", [
    (dict(batch=-1), INVALID), (dict(tokens=-1), INVALID), (dict(k_new=None), INVALID), (dict(start=None), INVALID),
    (dict(page_table=None), INVALID), (dict(max_pages=-1), INVALID), (dict(table_stride=-4), INVALID),
    (dict(v_new=PTR + 2), INVALID), (dict(k_new_stride=(128, 60, 128)), INVALID),
    (dict(v_new_stride=(128, 64, -128), tokens=2), INVALID), (dict(batch=65536), UNSUPPORTED),
    (dict(max_pages=1 << 30), UNSUPPORTED), (dict(tokens=(1 << 30) + 1), UNSUPPORTED)])
def test_append_refusals(gae, bad, status):
    _refused(gae, "gae_paged_append", gae.PagedAppendArgs, APPEND, bad, status)


@pytest.mark.parametrize("bad,status", [
    (dict(batch=-1), INVALID), (dict(heads=0), INVALID), (dict(heads=3), INVALID), (dict(q=None), INVALID),
    (dict(o=PTR + 8), INVALID), (dict(seq_lens=None), INVALID), (dict(q_stride=(256, 60)), INVALID),
    (dict(o_stride=(256, -64)), INVALID), (dict(scale=-1.0), UNSUPPORTED), (dict(scale=float("nan")), UNSUPPORTED),
    (dict(weights=PTR), INVALID), (dict(weights_out=PTR), INVALID),
    (dict(weights=PTR, weights_out=PTR, weights_len=63), INVALID),
    (dict(weights=PTR, weights_out=PTR, weights_len=64, w_stride=(-1, 0)), INVALID),
    (dict(weights=PTR, weights_out=PTR, weights_len=64, workspace_bytes=16), INVALID),
    (dict(weights=PTR, weights_out=PTR, weights_len=64, workspace=None), INVALID),
    (dict(o_stride=(256, 0)), INVALID), (dict(batch=2, o_stride=(0, 64)), INVALID),
    (dict(weights=PTR, weights_out=PTR, weights_len=64, w_out_stride=(64, 0)), INVALID),
    (dict(batch=65536), UNSUPPORTED)])
def test_attention_refusals(gae, bad, status):
    _refused(gae, "gae_paged_attn_fwd", gae.PagedAttnArgs, ATTN, bad, status)


@pytest.mark.parametrize("bad,status", [
    (dict(batch=0), INVALID), (dict(heads=3), INVALID), (dict(kv_heads=0), INVALID), (dict(seq_q=-1), INVALID),
    (dict(head_dim=96), UNSUPPORTED), (dict(dtype=0), UNSUPPORTED), (dict(q=None), INVALID), (dict(out=None), INVALID),
    (dict(k=PTR + 8), INVALID), (dict(k_stride=(4096, 1024, 60)), INVALID), (dict(lse_stride=(-1, 16)), INVALID),
    (dict(scale=-0.5), UNSUPPORTED), (dict(batch=20000), UNSUPPORTED),
    (dict(out_stride=(32, 0)), INVALID), (dict(workspace_bytes=0, workspace=None, seq_q=1 << 16), INVALID)])
def test_key_weights_refusals(gae, bad, status):
    a = _args(gae.KeyWeightsArgs, KEYS, **bad)
    assert gae.lib().gae_key_weights(C.byref(a), None) == status


@pytest.mark.parametrize("bad,status", [
    (dict(batch=-1), INVALID), (dict(keep=0), INVALID), (dict(recent=-1), INVALID), (dict(recent=33), INVALID),
    (dict(keep=33), INVALID), (dict(dst_table=PTR), INVALID), (dict(weights=None), INVALID), (dict(kept=None), INVALID),
    (dict(seq_lens=None), INVALID), (dict(w_stride=(-1, 0)), INVALID), (dict(weights_len=-1), INVALID),
    (dict(dst_table=None), INVALID), (dict(batch=65536), UNSUPPORTED), (dict(new_lens=PTR, seq_lens=PTR), INVALID),
    (dict(kept_weights=PTR, weights=PTR), INVALID)])
def test_evict_refusals(gae, bad, status):
    _refused(gae, "gae_paged_evict", gae.PagedEvictArgs, EVICT, bad, status)


def test_null_structs(gae):
    L, pool = gae.lib(), _pool(gae)
    for fn in ("gae_paged_append", "gae_paged_attn_fwd", "gae_paged_evict"):
        assert getattr(L, fn)(None, None, None) == INVALID
        assert getattr(L, fn)(C.byref(pool), None, None) == INVALID
    assert L.gae_key_weights(None, None) == INVALID


def test_empty_calls_touch_nothing(gae):
    L, pool = gae.lib(), _pool(gae)
    for fn, cls, base in (("gae_paged_append", gae.PagedAppendArgs, APPEND),
                          ("gae_paged_attn_fwd", gae.PagedAttnArgs, ATTN),
                          ("gae_paged_evict", gae.PagedEvictArgs, EVICT)):
        assert getattr(L, fn)(C.byref(pool), C.byref(_args(cls, base, batch=0)), None) == 0
    assert L.gae_paged_append(C.byref(pool), C.byref(_args(gae.PagedAppendArgs, APPEND, tokens=0)), None) == 0
    assert L.gae_key_weights(C.byref(_args(gae.KeyWeightsArgs, KEYS, seq_kv=0)), None) == 0


def test_python_refusals(gae):
    """The wrappers' own checks, on CPU tensors: shapes and types first, the device last."""
    z = torch.zeros
    k = z(4, 2, 16, 64, dtype=torch.bfloat16)
    table, ints = z(3, 2, dtype=torch.int32), z(3, dtype=torch.int32)
    new = z(3, 2, 5, 64, dtype=torch.bfloat16)
    q = z(3, 4, 64, dtype=torch.bfloat16)
    w = z(3, 2, 32)
    append = lambda **s: gae.paged_append(**{**dict(k_new=new, v_new=new, k_pages=k, v_pages=k, page_table=table,  # noqa: E731
                                                    start=ints), **s})
    attend = lambda **s: gae.paged_attention(**{**dict(q=q, k_pages=k, v_pages=k, page_table=table,  # noqa: E731
                                                       seq_lens=ints), **s})
    evict = lambda **s: gae.paged_evict(**{**dict(k_pages=k, v_pages=k, page_table=table, seq_lens=ints, weights=w,  # noqa: E731
                                                  dst_table=z(3, 1, dtype=torch.int32), keep=8), **s})
    keys = lambda **s: gae.attention_key_weights(**{**dict(q=z(1, 2, 8, 64), k=z(1, 2, 8, 64), lse=z(1, 2, 8)), **s})  # noqa: E731
    calls = [
        lambda: append(k_new=new.float()), lambda: append(v_new=new[:, :, :3]), lambda: append(k_new=new[0]),
        lambda: append(start=ints.long()), lambda: append(counts=ints[:2]), lambda: append(page_table=table.long()),
        lambda: append(page_table=table[:2]), lambda: append(v_pages=k[:3]), lambda: append(k_pages=k.transpose(2, 3)),
        lambda: append(k_new=z(3, 3, 5, 64, dtype=torch.bfloat16), v_new=z(3, 3, 5, 64, dtype=torch.bfloat16)),
        lambda: attend(q=q[0]), lambda: attend(q=q.float()), lambda: attend(q=q[..., :32]),
        lambda: attend(seq_lens=ints[:1]), lambda: attend(weights=w[..., :31]), lambda: attend(weights_out=w),
        lambda: attend(weights=w.double()), lambda: attend(lse=z(3, 3)), lambda: attend(out=q.float()),
        lambda: attend(page_table=table.t()),
        lambda: evict(weights=w[:, :1]), lambda: evict(dst_table=z(2, 1, dtype=torch.int32)),
        lambda: evict(seq_lens=ints.float()),
        lambda: keys(q=z(2, 8, 64)), lambda: keys(k=z(1, 2, 8, 32)), lambda: keys(lse=z(1, 2, 7)),
        lambda: keys(accumulate=True), lambda: keys(out=z(1, 2, 7)),
        # all in order but for the device
        append, attend, evict, keys,
    ]
    for i, call in enumerate(calls):
        with pytest.raises(gae.GAEError):
            call()
            pytest.fail(f"call {i} was accepted")


def test_cache_refusals(gae):
    """PagedKVCache's own bookkeeping, on CPU tensors: nothing is launched."""
    new = lambda **kw: gae.PagedKVCache(1, 2, 2, 64, 40, page_size=16, device="cpu", **kw)  # noqa: E731
    for bad in (dict(budget=0), dict(budget=41), dict(budget=8, recent=9)):
        with pytest.raises(gae.GAEError):
            new(**bad)
    c = new()
    assert c.table.shape == (2, 3) and c.table.unique().numel() == 6 and c.spare is None
    k = torch.zeros(2, 2, 1, 64, dtype=torch.bfloat16)
    for call in (lambda: c.append(0, k, k), c.commit, c.evict, lambda: c.reserve(41), lambda: c.reserve(3, [1]),
                 lambda: c.reserve(3, [1, 4])):
        with pytest.raises(gae.GAEError):
            call()
    c.reserve(30, [30, 7])
    c.commit()
    assert c.lengths == [30, 7] and c.lens.tolist() == [30, 7]
    with pytest.raises(gae.GAEError):  # 30 + 11 > 40
        c.reserve(11)
    b = new(budget=20, recent=4)
    assert b.spare.shape == (2, 2) and not set(b.spare.flatten().tolist()) & set(b.table.flatten().tolist())
    b.reserve(20)
    with pytest.raises(gae.GAEError):  # between reserve and commit
        b.evict()
    b.commit()
    assert b.evict() is None
    with pytest.raises(gae.GAEError):  # not empty any more
        gae.layer_stack_prefill([], torch.zeros(2, 1, 128, dtype=torch.bfloat16), b)


def _cpu_cache(gae, **kw):
    return gae.PagedKVCache(1, 2, 2, 64, 40, page_size=16, device="cpu", **kw)


@pytest.mark.parametrize("counts", [None, [3, 1]])
@pytest.mark.parametrize("given", [0, 1, 2, 4])
def test_cache_append_takes_the_tokens_reserved(gae, counts, given):
    """Fewer tokens than reserved would leave positions that no one wrote."""
    c = _cpu_cache(gae)
    c.reserve(3, counts)
    k = torch.zeros(2, 2, given, 64, dtype=torch.bfloat16)
    with pytest.raises(gae.GAEError, match=f"append of {given} tokens, 3 reserved"):
        c.append(0, k, k)


def test_cache_prompt_weights_take_the_tokens_reserved(gae):
    c = _cpu_cache(gae, budget=20)
    q = torch.zeros(2, 2, 3, 64, dtype=torch.bfloat16)
    lse = torch.zeros(2, 2, 3)
    with pytest.raises(gae.GAEError, match="prompt weights without reserve"):
        c.add_prompt_weights(0, q, q, lse)
    c.reserve(4)
    for qq, kk in ((q, q), (torch.cat([q, q[:, :, :1]], 2), q)):
        with pytest.raises(gae.GAEError, match="4 tokens reserved"):
            c.add_prompt_weights(0, qq, kk, lse)


def test_cache_reserves_no_negative_tokens(gae):
    c = _cpu_cache(gae)
    c.reserve(7)
    c.commit()
    for counts in (None, [0, 0], [-5, -5]):
        with pytest.raises(gae.GAEError):
            c.reserve(-5, counts)
    assert c.lengths == [7, 7] and c.next_lens.tolist() == [7, 7]


def test_cache_refresh_tells_of_lost_tokens(gae):
    c = _cpu_cache(gae)
    c.lens.copy_(torch.tensor([40, 3]))
    c.refresh()
    assert c.lengths == [40, 3]
    c.lens.copy_(torch.tensor([3, 41]))
    with pytest.raises(gae.GAEError, match="41 positions, room for 40"):
        c.refresh()


def test_python_refusals_name_their_reason(gae):
    """Each check of the wrappers by the words of its own refusal: a call that slipped through one would
    end at the device check, whose words are others."""
    z = torch.zeros
    half = dict(dtype=torch.bfloat16)
    k = z(4, 2, 16, 64, **half)
    table, ints = z(3, 2, dtype=torch.int32), z(3, dtype=torch.int32)
    new, q, w = z(3, 2, 5, 64, **half), z(3, 4, 64, **half), z(3, 2, 32)
    wide = z(3, 4, dtype=torch.int32)

    def call(fn, base, **s):
        return lambda: fn(**{**base, **s})

    append = lambda **s: call(gae.paged_append, dict(k_new=new, v_new=new, k_pages=k, v_pages=k, page_table=table,  # noqa: E731
                                                     start=ints), **s)
    attend = lambda **s: call(gae.paged_attention, dict(q=q, k_pages=k, v_pages=k, page_table=table, seq_lens=ints), **s)  # noqa: E731
    evict = lambda **s: call(gae.paged_evict, dict(k_pages=k, v_pages=k, page_table=table, seq_lens=ints, weights=w,  # noqa: E731
                                                   dst_table=z(3, 1, dtype=torch.int32), keep=8), **s)
    keys = lambda **s: call(gae.attention_key_weights, dict(q=z(1, 2, 8, 64), k=z(1, 2, 8, 64), lse=z(1, 2, 8)), **s)  # noqa: E731
    for c, why in [
        (append(k_new=new.float(), v_new=new.float()), "new rows and pages must share a dtype"),
        (append(v_new=new.float()), "new rows and pages must share a dtype"),
        (append(v_new=new[:, :, :3]), r"must be \[batch, kv_heads, tokens, head_dim\]"),
        (append(k_new=new[0], v_new=new[0]), r"must be \[batch, kv_heads, tokens, head_dim\]"),
        (append(k_new=z(3, 3, 5, 64, **half), v_new=z(3, 3, 5, 64, **half)), "differ in heads or head_dim"),
        (append(k_new=new[..., :32], v_new=new[..., :32]), "differ in heads or head_dim"),
        (append(k_new=z(3, 2, 64, 5, **half).transpose(2, 3)), "new rows must have a contiguous head_dim"),
        (append(start=ints.long()), r"start must be contiguous int32 \[batch\]"),
        (append(start=z(6, dtype=torch.int32)[::2]), r"start must be contiguous int32 \[batch\]"),
        (append(counts=ints[:2]), r"counts must be contiguous int32 \[batch\]"),
        (append(counts=ints.float()), r"counts must be contiguous int32 \[batch\]"),
        (append(page_table=table.long()), r"page_table must be int32 \[batch, max_pages\]"),
        (append(page_table=table[:2]), r"page_table must be int32 \[batch, max_pages\]"),
        (append(page_table=table[0]), r"page_table must be int32 \[batch, max_pages\]"),
        (append(page_table=wide[:, ::2]), "page_table must have contiguous rows"),
        (append(v_pages=k[:3]), r"must be \[num_pages, kv_heads, page_size, head_dim\]"),
        (append(k_pages=k[0], v_pages=k[0]), r"must be \[num_pages, kv_heads, page_size, head_dim\]"),
        (append(v_pages=k.half()), "k_pages and v_pages must share a dtype"),
        (append(k_pages=z(4, 2, 64, 16, **half).transpose(2, 3)), "pages must have a contiguous head_dim"),
        (append(k_pages=k.long(), v_pages=k.long()), "unsupported dtype"),
        (attend(q=q[0]), r"q must be \[batch, heads, head_dim\]"),
        (attend(q=q.float()), "differ in head_dim or dtype"),
        (attend(q=q[..., :32]), "differ in head_dim or dtype"),
        (attend(q=z(3, 64, 4, **half).transpose(1, 2)), "q must have a contiguous head_dim"),
        (attend(seq_lens=ints[:1]), r"seq_lens must be contiguous int32 \[batch\]"),
        (attend(seq_lens=ints.long()), r"seq_lens must be contiguous int32 \[batch\]"),
        (attend(page_table=wide[:, ::2]), "page_table must have contiguous rows"),
        (attend(page_table=table.t()), r"page_table must be int32 \[batch, max_pages\]"),
        (attend(weights=w[..., :31]), r"weights must be fp32 \[3, 2, >= 32\]"),
        (attend(weights=w.double()), r"weights must be fp32 \[3, 2, >= 32\]"),
        (attend(weights=w[:, :1]), r"weights must be fp32 \[3, 2, >= 32\]"),
        (attend(weights=z(3, 2, 64)[..., ::2]), "weights must have contiguous rows"),
        (attend(weights=w, weights_out=w[..., :31]), r"weights_out must be fp32 \[3, 2, >= 32\]"),
        (attend(weights_out=w), "weights_out without weights"),
        (attend(lse=z(3, 3)), r"lse must be contiguous fp32 \[batch, heads\]"),
        (attend(lse=z(4, 3).t()), r"lse must be contiguous fp32 \[batch, heads\]"),
        (attend(lse=z(3, 4, **half)), r"lse must be contiguous fp32 \[batch, heads\]"),
        (attend(out=q.float()), "out must be like q"),
        (attend(out=q[:2]), "out must be like q"),
        (attend(out=z(3, 64, 4, **half).transpose(1, 2)), "out must be like q"),
        (evict(weights=w[:, :1]), r"weights must be fp32 \[3, 2, >= 0\]"),
        (evict(weights=w.half()), r"weights must be fp32 \[3, 2, >= 0\]"),
        (evict(dst_table=z(2, 1, dtype=torch.int32)), r"dst_table must be int32 \[batch, max_pages\]"),
        (evict(seq_lens=ints.float()), r"seq_lens must be contiguous int32 \[batch\]"),
        (evict(keep=0), "keep must be positive"),
        (keys(q=z(2, 8, 64)), r"must be \[batch, heads, seq, head_dim\]"),
        (keys(k=z(1, 2, 8, 32)), "differ in batch, head_dim or dtype"),
        (keys(k=z(1, 2, 8, 64).half()), "differ in batch, head_dim or dtype"),
        (keys(k=z(2, 2, 8, 64)), "differ in batch, head_dim or dtype"),
        (keys(q=z(1, 2, 64, 8).transpose(2, 3)), "q and k must have a contiguous head_dim"),
        (keys(lse=z(1, 2, 7)), r"lse must be fp32 \[1, 2, >= 8\]"),
        (keys(lse=z(1, 2, 9)), r"lse must be \[batch, heads, seq_q\]"),
        (keys(lse=z(1, 2, 16)[..., ::2]), "lse must have contiguous rows"),
        (keys(accumulate=True), "accumulate needs out"),
        (keys(out=z(1, 2, 7)), r"out must be \[1, 2, 8\]"),
        # all in order but for the device
        (append(), "k_pages is on cpu"), (append(counts=ints), "k_pages is on cpu"), (attend(), "q is on cpu"),
        (attend(weights=w), "q is on cpu"), (evict(), "k_pages is on cpu"), (keys(), "q is on cpu"),
    ]:
        with pytest.raises(gae.GAEError, match=why):
            c()


def test_key_weights_query_tiles_fit_an_int(gae):
    """2^23 query tiles times 256 heads on one key head are 2^31: one too many."""
    L, n = gae.lib(), 1 << 30
    wide = dict(heads=256, kv_heads=1, seq_q=n, q_stride=(0, 0, 64), lse_stride=(0, 0), out_stride=(16, 16))
    assert L.gae_key_weights(C.byref(_args(gae.KeyWeightsArgs, KEYS, **wide)), None) == UNSUPPORTED
    assert b"query tiles" in _last_error(L)


def _last_error(L):
    buf = C.create_string_buffer(512)
    L.gae_last_error(buf, 512)
    return buf.value


def test_layer_refuses_what_does_not_fit_it(gae):
    """Before a kernel reads a row as wide as x from parameters of another width, or a row is written."""
    z = lambda *s, t=torch.bfloat16: torch.zeros(*s, dtype=t)  # noqa: E731
    layer = gae.Gpt2Layer.random(256, 4, 512, device="cpu")
    new = lambda heads=4, hd=64, t=torch.bfloat16: gae.PagedKVCache(1, 2, heads, hd, 40, dtype=t, device="cpu")  # noqa: E731
    for x, cache, i, why in [
        (z(2, 512), new(), 0, r"x must be bf16 \[2, 256\]"), (z(2, 255), new(), 0, r"x must be bf16 \[2, 256\]"),
        (z(3, 256), new(), 0, r"x must be bf16 \[2, 256\]"), (z(256), new(), 0, r"x must be bf16 \[2, 256\]"),
        (z(2, 256, t=torch.float32), new(), 0, r"x must be bf16 \[2, 256\]"),
        (z(2, 256), new(), 1, "layer 1 of a cache of 1"), (z(2, 256), new(2), 0, "4 heads of 64"),
        (z(2, 256), new(4, 32), 0, "4 heads of 64"), (z(2, 256), new(t=torch.float16), 0, "4 heads of 64"),
        (z(2, 256), new(), 0, "x must be on the current CUDA device"),
    ]:
        cache.reserve(1)
        with pytest.raises(gae.GAEError, match=why):
            layer.decode(x, cache, i)
        with pytest.raises(gae.GAEError, match=why.replace("[2, 256", "[2, S, 256")):
            layer.prefill(x.unsqueeze(1), cache, i)
