"""What the operators of a serving step refuse, before anything is launched: on the CPU, through the C ABI and through the operators."""
import pytest
import torch

F32, F16, BF16 = 0, 1, 2


def test_rope_and_append_refusals(xn):
    lib = xn.lib()

    def rope(dtype=BF16, dst=16, src=16, pos=16, freqs=16, tokens=2, heads=2, hd=64, rot=64):
        return lib.xn_mm_rope(dtype, dst, heads * hd, hd, src, heads * hd, hd, pos, freqs, tokens, heads, hd, rot, 0, None)

    assert rope(dtype=5) == 1 and rope(hd=63) == 1 and rope(rot=66) == 1 and rope(rot=7) == 1
    assert rope(dst=None) == 1 and rope(src=None) == 1 and rope(pos=None) == 1 and rope(freqs=None) == 1
    assert b"null" in lib.xn_mm_last_error()
    assert rope(tokens=0, dst=None) == 0 and rope(heads=0, dst=None) == 0 and rope(hd=0, rot=0, dst=None) == 0
    assert rope(tokens=2 ** 40) == 1

    def append(dtype=BF16, kp=16, vp=16, pages=4, page=16, k=16, v=16, slots=16, tokens=2, kv=2, hd=64, qd=None, q=None, heads=0, pos=16,
               freqs=16, rot=64):
        return lib.xn_mm_paged_append(dtype, kp, vp, kv * page * hd, page * hd, hd, pages, page, k, kv * hd, hd, v, kv * hd, hd, slots,
                                      tokens, kv, hd, qd, q, heads * hd, hd, heads, pos, freqs, rot, 0, None)

    assert append(dtype=-1) == 1 and append(page=0) == 1 and append(hd=63, rot=0) == 1 and append(rot=128) == 1
    for missing in ("kp", "vp", "k", "v", "slots", "pos"):
        assert append(**{missing: None}) == 1, missing
    assert append(qd=16, q=None, heads=4) == 1
    assert append(tokens=0, kp=None) == 0


def test_attention_paged_refusals(xn):
    lib = xn.lib()
    need = lib.xn_mm_attention_paged_workspace_bytes(128)
    assert need > 0 and lib.xn_mm_attention_paged_workspace_bytes(96) == 0

    def call(dtype=BF16, out=16, q=16, tokens=4, heads=8, kp=16, vp=16, pages=8, page=16, kv=2, hd=128, table=16, ts=4, mp=4, ctx=16,
             starts=16, batch=2, mq=0, window=0, scale=0.1, ws=256, wsb=None, qt=None, ps=None):
        return lib.xn_mm_attention_paged(dtype, out, heads * hd, hd, q, heads * hd if qt is None else qt, hd, tokens, heads, kp, vp,
                                         kv * page * hd if ps is None else ps, page * hd, hd, pages, page, kv, hd, table, ts, mp, ctx,
                                         starts, batch, mq, window, scale, ws, need if wsb is None else wsb, None)

    assert call(dtype=F32) == 1 and b"16-bit" in lib.xn_mm_last_error()
    assert call(hd=96) == 1 and b"head_dim" in lib.xn_mm_last_error()
    assert call(heads=9) == 1 and call(kv=0) == 1
    for bad in (-0.5, float("nan"), float("inf")):
        assert call(scale=bad) == 1 and b"scale" in lib.xn_mm_last_error()
    assert call(page=0) == 1 and call(mp=2 ** 30) == 1 and call(tokens=2 ** 31) == 1
    assert call(tokens=0, out=None) == 0 and call(batch=0, out=None) == 0
    assert call(starts=None) == 1  # four rows for two sequences
    for missing in ("out", "q", "ctx", "table", "kp", "vp"):
        assert call(**{missing: None}) == 1 and b"null" in lib.xn_mm_last_error(), missing
    assert call(q=24) == 1 and call(kp=8) == 1 and call(out=2) == 1 and call(qt=8 * 128 + 4) == 1 and call(ps=2 * 16 * 128 + 1) == 1
    assert b"aligned" in lib.xn_mm_last_error()
    assert call(ws=None) == 4 and call(wsb=need - 1) == 4 and call(ws=128) == 1


def test_sample_refusals(xn):
    lib = xn.lib()

    def call(dtype=F32, out=16, x=16, rows=2, vocab=100, u=16):
        return lib.xn_mm_sample(dtype, out, x, vocab, rows, vocab, u, None, None, None, None, None)

    assert call(dtype=4) == 1 and call(vocab=0) == 1 and call(vocab=2 ** 20 + 1) == 1 and call(x=18) == 1
    assert call(out=None) == 1 and call(x=None) == 1 and call(u=None) == 1
    assert call(rows=0, out=None) == 0


def test_operators_refuse_shapes_and_types(xn):
    bf, f64, i64, i32 = torch.bfloat16, torch.float64, torch.int64, torch.int32
    x, pos, fr = torch.zeros(3, 4, 64, dtype=bf), torch.zeros(3, dtype=i64), torch.zeros(32, dtype=f64)
    for args in ((x.double(), pos, fr), (x[0], pos, fr), (x, pos[:2], fr), (x, pos.int(), fr), (x, pos, fr.float()),
                 (x, pos, torch.zeros(33, dtype=f64)), (x[..., :63], pos, fr[:3])):
        with pytest.raises(xn.XnError):
            xn.rope(*args)
    with pytest.raises(xn.XnError, match="broadcast"):
        xn.rope(x, pos, fr, out=x[:1].expand(3, 4, 64))
    with pytest.raises(xn.XnError, match="CUDA tensors only"):
        xn.rope(x, pos, fr)

    kp, vp, k = torch.zeros(5, 2, 16, 64, dtype=bf), torch.zeros(5, 2, 16, 64, dtype=bf), torch.zeros(3, 2, 64, dtype=bf)
    ok = dict(k_pages=kp, v_pages=vp, k=k, v=k, slots=pos, q=x, positions=pos, freqs=fr)
    for bad in (dict(k_pages=kp[0]), dict(v_pages=vp[:4]), dict(v_pages=vp.half()), dict(v_pages=vp.transpose(1, 2).contiguous().transpose(1, 2)),
                dict(k=k[:2]), dict(v=k[:, :1]), dict(k=k.float()), dict(slots=pos.int()), dict(q=x[:2]), dict(q=x[..., :32]),
                dict(positions=None), dict(freqs=None), dict(freqs=torch.zeros(40, dtype=f64)),
                dict(k_pages=kp[:1].expand(5, 2, 16, 64), v_pages=vp[:1].expand(5, 2, 16, 64))):
        with pytest.raises(xn.XnError):
            xn.paged_append_(**{**ok, **bad})
    with pytest.raises(xn.XnError, match="CUDA tensors only"):
        xn.paged_append_(**ok)

    table, ctx, st = torch.zeros(2, 4, dtype=i32), torch.zeros(2, dtype=i32), torch.zeros(3, dtype=i32)
    ok = dict(q=x, k_pages=kp, v_pages=vp, page_table=table, context=ctx, scale=0.1, query_starts=st)
    for bad in (dict(q=x.float()), dict(q=x[0]), dict(q=x[:, :3]), dict(k_pages=kp[..., :32], v_pages=vp[..., :32]), dict(k_pages=kp.half()),
                dict(page_table=table.long()), dict(page_table=table[0]), dict(context=ctx[:1]), dict(query_starts=st[:2]),
                dict(query_starts=None), dict(window=-1), dict(max_query=-1), dict(out=x[:2]), dict(out=x.float())):
        with pytest.raises(xn.XnError):
            xn.attention_paged(**{**ok, **bad})
    with pytest.raises(xn.XnError, match="CUDA tensors only"):
        xn.attention_paged(**ok)

    lg, u = torch.zeros(2, 50), torch.zeros(2)
    for args, kw in (((lg.double(), u), {}), ((lg[0], u), {}), ((lg, u[:1]), {}), ((lg, u.double()), {}), ((lg[:, :0], u), {}),
                     ((lg, u), dict(top_k=u)), ((lg, u), dict(temperature=u.double())), ((lg, u), dict(top_p=u[:1])),
                     ((lg, u), dict(min_p=u.int()))):
        with pytest.raises(xn.XnError):
            xn.sample(*args, **kw)
    with pytest.raises(xn.XnError, match="CUDA tensors only"):
        xn.sample(lg, u)
