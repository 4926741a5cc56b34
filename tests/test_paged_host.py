"""Paged caches and token log probabilities without a device: what the entry points refuse (before anything is launched), the layouts of
their descriptors, and the contracts of indexes outside their range, restated in oracle/kernel_emulation.py."""
import ctypes as C

import pytest
import torch

from neurst_amd import _lib
from neurst_amd import kernels as K
from oracle import kernel_emulation as E

L = _lib.lib
ARG, NOWHERE = -1, C.c_void_p(4096)


def message():
    return L.nst_last_error_string().decode()


def i32(a):
    return torch.tensor(a, dtype=torch.int32)


def test_descriptor_layouts():
    assert C.sizeof(_lib.NstPagedPool) == 64 and C.sizeof(_lib.NstPagedAttnDesc) == 136
    for f in _lib.NstPagedPool._fields_:
        if f[0] != "reserved":
            assert getattr(_lib.NstPagedAttnDesc, f[0]).offset == 72 + getattr(_lib.NstPagedPool, f[0]).offset


def plan(B=1, stride=4, max_pages=4, n_free=1, page_size=4, max_tokens=1, cursor_out=8192, seq=12288, free=4096, slots=4096, cached=4096):
    return L.nst_paged_plan(cached, 4096, B, 4096, stride, max_pages, free, n_free, 4096, page_size, slots, max_tokens, seq, 16384, cursor_out, None)


@pytest.mark.parametrize("kw,text", [
    (dict(B=-1), "B=-1"), (dict(page_size=0), "page_size=0"), (dict(max_pages=0), "max_pages=0"), (dict(max_tokens=-1), "max_tokens=-1"),
    (dict(stride=3), "stride 3"), (dict(max_pages=1 << 20, stride=1 << 20, page_size=1 << 12), "2^30"), (dict(slots=None), "NULL"),
    (dict(free=None), "NULL"), (dict(cached=None), "NULL"), (dict(cursor_out=4096), "overlap"), (dict(seq=4096), "overlap")])
def test_plan_refuses(kw, text):
    assert plan(**kw) == ARG and text in message()


def attn(**kw):
    d = _lib.NstPagedAttnDesc(2, 4, 2, 64, 4, 0, 0.125, 0, 256, 64, 256, 64, 4, 8, 16, _lib.NST_BF16, 0, 1024, 64, 64, 1024, 64, 64)
    ptr = dict(q=4096, k=4096, v=4096, table=4096, lens=4096, out=4096)
    for n, v in kw.items():
        if n in ptr:
            ptr[n] = v
        else:
            setattr(d, n, v)
    rc = L.nst_paged_attention(C.byref(d), ptr["q"], ptr["k"], ptr["v"], ptr["table"], ptr["lens"], ptr["out"], None, None, 0, None)
    return rc, d


@pytest.mark.parametrize("kw,text", [
    (dict(H=3), "3 heads over 2"), (dict(Hkv=0), "0 key"), (dict(dh=257), "head size 257"), (dict(dh=0), "head size 0"), (dict(dtype=2), "dtype 2"),
    (dict(page_size=0), "page_size=0"), (dict(table_stride=3), "stride 3"), (dict(max_len=-1), "max_len=-1"), (dict(q=None), "NULL"),
    (dict(k=None), "NULL"), (dict(out=None), "NULL"), (dict(lens=None), "NULL"), (dict(max_pages=1 << 28, table_stride=1 << 28), "2^30"),
    (dict(B=1 << 30), "rows")])
def test_attention_refuses(kw, text):
    rc, d = attn(**kw)
    assert rc == ARG and text in message()
    if not {"q", "k", "out", "lens"} & set(kw):
        assert L.nst_paged_attention_workspace_bytes(C.byref(d)) == ARG
    assert L.nst_paged_attention(None, 1, 1, 1, 1, 1, 1, None, None, 0, None) == ARG


def test_empty_calls_launch_nothing():
    rc, _ = attn(B=0)
    assert rc == 0
    pool = _lib.NstPagedPool(8, 16, _lib.NST_F32, 0, 1024, 64, 64, 1024, 64, 64)
    assert L.nst_paged_append(None, None, 0, 1, 64, 64, 64, 64, 64, None, None, C.byref(pool), None, None) == 0
    assert L.nst_paged_append(None, None, 3, 1, 64, 64, 64, 64, 64, None, None, C.byref(pool), None, None) == ARG
    assert L.nst_token_logprobs_fwd(None, None, None, None, None, None, None, 0, 10, 10, 0, _lib.NST_F32, None, 0, None) == 0
    assert L.nst_token_logprobs_bwd(None, None, None, None, None, None, None, 0, 10, 10, 10, _lib.NST_F32, None) == 0


@pytest.mark.parametrize("args,text", [
    (dict(V=0), "V=0"), (dict(V=(1 << 20) + 1), "2^20"), (dict(top_n=65), "top_n=65"), (dict(V=5, top_n=6), "top_n=6"), (dict(top_n=-1), "top_n=-1"),
    (dict(dtype=3), "dtype 3"), (dict(rows=-1), "rows=-1"), (dict(logits=None), "NULL"), (dict(top_ids=None), "NULL"), (dict(tokens=None), "NULL")])
def test_token_logprobs_refuses(args, text):
    a = dict(logits=4096, tokens=4096, top_ids=4096, rows=2, V=100, ldl=100, top_n=3, dtype=_lib.NST_F32)
    a.update(args)
    rc = L.nst_token_logprobs_fwd(a["logits"], a["tokens"], 4096, 4096, 4096, 4096, a["top_ids"], a["rows"], a["V"], a["ldl"], a["top_n"], a["dtype"],
                                  None, 0, None)
    assert rc == ARG and text in message()


def test_token_logprobs_gradient_refuses():
    def bwd(lse=4096, dlogp=4096, tokens=4096, dent=None, ent=None, out=8192, ldl=10, ldd=10, rows=2):
        return L.nst_token_logprobs_bwd(4096, tokens, lse, ent, dlogp, dent, out, rows, 10, ldl, ldd, _lib.NST_F32, None)
    for kw in (dict(lse=None), dict(out=None), dict(tokens=None), dict(dent=4096), dict(ldd=9), dict(out=4096, ldd=12)):
        assert bwd(**kw) == ARG, kw


def reorder(planes=2, plane=4096, pages=4, page=1024, ps=4, tok=256, tin=4096, ins=4, tout=8192, outs=4, W=4, rows=2, sin=4096, sout=8192, pool=4096):
    return L.nst_paged_reorder(pool, planes, plane, pages, page, ps, tok, tin, ins, tout, outs, W, rows, 4096, 4096, sin, sout, None)


@pytest.mark.parametrize("kw,text", [
    (dict(planes=0), "planes=0"), (dict(planes=1 << 17), "planes"), (dict(ps=0), "page_size=0"), (dict(page=1023), "apart"), (dict(ins=3), "strides"),
    (dict(outs=3), "strides"), (dict(tout=4096), "overlap"), (dict(sout=4096), "overlap"), (dict(pool=None), "NULL"), (dict(rows=-1), "rows=-1")])
def test_reorder_refuses(kw, text):
    assert reorder(**kw) == ARG and text in message()


def test_wrappers_refuse_shapes_types_and_host_tensors():
    pool = torch.zeros(4, 16, 2, 64)
    q, table, lens = torch.zeros(3, 4, 64), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        K.paged_attention(q, pool, pool, table, lens)
    with pytest.raises(ValueError, match="seq_lens"):
        K.paged_attention(q, pool, pool, table, lens.long())
    with pytest.raises(ValueError, match="seq_lens"):
        K.paged_attention(q, pool, pool, table, lens[:2])
    with pytest.raises(ValueError, match="block_table"):
        K.paged_attention(q, pool, pool, table[:2], lens)
    with pytest.raises(ValueError, match="block_table"):
        K.paged_attention(q, pool, pool, table.expand(3, 2).t().contiguous().t(), lens)
    with pytest.raises(ValueError, match="q "):
        K.paged_attention(q[..., :32], pool, pool, table, lens)
    with pytest.raises(ValueError, match="k_pool"):
        K.paged_attention(q, pool, pool.bfloat16(), table, lens)
    with pytest.raises(ValueError, match="dense"):
        K.paged_attention(q, pool.transpose(2, 3).contiguous().transpose(2, 3), pool, table, lens)
    with pytest.raises(TypeError, match="dtype"):
        K.paged_attention(q.half(), pool.half(), pool.half(), table, lens)
    with pytest.raises(ValueError, match="slots"):
        K.paged_append(q[:, :2], q[:, :2], pool, pool, torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="rows"):
        K.paged_append(q, q, pool, pool, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="new_lens"):
        K.paged_plan(lens, lens[:2], table, lens, lens[:1], 16, 4)
    with pytest.raises(ValueError, match="cursor"):
        K.paged_plan(lens, lens, table, lens, lens, 16, 4)
    with pytest.raises(ValueError, match="parents"):
        K.paged_reorder(torch.zeros(2, 4, 16, 8), table, lens, lens, lens)
    with pytest.raises(ValueError, match="dense pages"):
        K.paged_reorder(torch.zeros(2, 4, 16, 8).transpose(1, 2), table, lens, lens.long(), lens)
    with pytest.raises(ValueError, match="tokens"):
        K.token_logprobs(torch.zeros(3, 5), lens)
    with pytest.raises(ValueError, match="logits"):
        K.token_logprobs(torch.zeros(5, 3).t(), lens.long())
    with pytest.raises(ValueError, match="out"):
        K.token_logprobs_bwd(torch.zeros(3, 5), lens.long(), torch.zeros(3), torch.zeros(3), torch.zeros(3), out=torch.zeros(3, 6))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        K.token_logprobs(torch.zeros(3, 5), lens.long())


# ------------------------------------------------------------------------------------------------ contracts
def test_plan_contract_when_pages_run_out():
    table = torch.full((3, 3), -1, dtype=torch.int32)
    table[0, 0] = 9
    slots, lens, cu, cursor = E.paged_plan(i32([2, 0, 0]), i32([4, 3, 5]), table, i32([5, 6]), i32([0]), 4, 14)
    # request 0: tokens 2, 3 in page 9, 4, 5 in page 5; request 1 gets page 6; request 2 gets nothing
    assert slots.tolist() == [38, 39, 20, 21, 24, 25, 26] + [-1] * 7
    assert lens.tolist() == [6, 3, 0] and cu.tolist() == [0, 4, 7, 12] and cursor.tolist() == [2]
    assert table.tolist() == [[9, 5, -1], [6, -1, -1], [-1, -1, -1]]


def test_plan_contract_for_free_entries_that_name_no_page():
    """They count as pages, enter the table as -1 over whatever stood there, and give their tokens no slot."""
    table = i32([[3, 0, 7], [4, 6, 5]])
    slots, lens, cu, cursor = E.paged_plan(i32([4, 0]), i32([3, 6]), table, i32([-5, 8, -1]), i32([0]), 4, 10)
    assert table.tolist() == [[3, -1, 7], [8, -1, 5]]
    assert slots.tolist() == [-1] * 3 + [32, 33, 34, 35] + [-1] * 3 and lens.tolist() == [7, 6] and cu.tolist() == [0, 3, 9] and cursor.tolist() == [3]


def test_attention_contract_for_bad_pages():
    k = torch.randn(2, 2, 1, 8, generator=torch.Generator().manual_seed(0))
    q = torch.ones(3, 1, 8)
    out, lse = E.paged_attention(q, k, k, i32([[0, 7], [-1, -1], [1, 0]]), i32([4, 4, 3]), return_lse=True)
    ref = torch.softmax((k[0, :, 0] @ q[0, 0]) / 8 ** 0.5, 0) @ k[0, :, 0]
    assert torch.allclose(out[0, 0], ref) and float(out[1].abs().sum()) == 0 and float(lse[1]) == -float("inf")
    ref2 = torch.cat([k[1], k[0, :1]])[:, 0]
    assert torch.allclose(out[2, 0], torch.softmax((ref2 @ q[2, 0]) / 8 ** 0.5, 0) @ ref2)


def test_reorder_contract():
    pool = torch.arange(6 * 4, dtype=torch.float32).view(1, 6, 4, 1)
    table, spare = i32([[0, -1], [1, -1]]), i32([4, 5])
    t, s = E.paged_reorder(pool, table, i32([3, 3]), torch.tensor([1, 1]), spare)
    assert t.tolist() == [[4, -1], [1, -1]] and s.tolist() == [0, 5]
    assert pool[0, 4, :, 0].tolist() == [4, 5, 6, 19] and pool[0, 0, :, 0].tolist() == [0, 1, 2, 3]
    t, s = E.paged_reorder(pool, table, i32([4, 4]), torch.tensor([1, 1]), spare)          # full pages are shared
    assert t.tolist() == [[1, -1], [1, -1]] and s.tolist() == [4, 5]
    t, s = E.paged_reorder(pool, table, i32([3, 2]), torch.tensor([1, 7]), spare)          # no such parent, another length
    assert t.tolist() == table.tolist() and s.tolist() == [4, 5]
