"""Host side of the token operators without a GPU: bucket borders, argument checks of the C entry points, refusal of CPU tensors."""
import ctypes
import math

import pytest
import torch


@pytest.mark.parametrize("nb,maxd,bi", [(32, 128, True), (32, 128, False), (16, 64, True), (64, 256, False), (8, 16, True), (4, 3, True), (64, 1024, True)])
def test_relative_buckets_rule(nb, maxd, bi):
    from diffusion_uncertainty_amd import ops
    b = ops.RelativeBuckets(nb, maxd, bi, device="cpu")
    m = b.map.tolist()
    assert len(m) == 2 * maxd + 1 and b.radius == maxd and min(m) == 0 and max(m) <= nb - 1
    side = nb // 2 if bi else nb
    ex = side // 2
    for rel in range(-maxd, maxd + 1):
        n = abs(rel) if bi else max(-rel, 0)
        if n < ex:
            want = n
        else:
            want = min(side - 1, ex + math.floor(math.log(n / ex) / math.log(maxd / ex) * (side - ex) + 1e-9))
        assert m[rel + maxd] == want + (side if bi and rel > 0 else 0), rel
    back = m[:maxd + 1][::-1]
    assert back == sorted(back) and back[maxd] == side - 1


def test_relative_buckets_refusals():
    from diffusion_uncertainty_amd import ops
    for a in [(1, 16, False), (2, 16, True), (7, 16, True), (32, 8, True), (32, 1025, True)]:
        with pytest.raises(ValueError):
            ops.RelativeBuckets(*a, device="cpu")
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.RelativeBuckets.from_map(torch.zeros(3, dtype=torch.int32), 4)


def test_no_cpu_fallback():
    from diffusion_uncertainty_amd import ops
    x = torch.zeros(2, 8)
    for call in (lambda: ops.sandwich_norm(x, x), lambda: ops.token_logprobs(x),
                 lambda: ops.rel_attention(x[None], x[None], x[None], x, None, heads=1)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def test_argument_validation_without_gpu():
    """Every refusal comes before a launch: no GPU is needed to see it."""
    from diffusion_uncertainty_amd import _lib
    L = _lib.lib()
    P = 4096

    def refuses(fn, args, text):
        assert fn(ctypes.byref(args), None) == -1
        assert text in L.dua_last_error().decode(), L.dua_last_error()

    def norm(**kw):
        a = _lib.SandwichNormArgs(x=P, y=P, rows=4, D=64, post=1, pre=1, res_scale=1.0, eps=1e-6, r=P, z=P, stats=P, dr=P, dz=P, dx=P, dy=P)
        for n, v in kw.items():
            setattr(a, n, v)
        return a

    assert L.dua_sandwich_norm(None, None) == -1 and L.dua_sandwich_norm_bwd(None, None) == -1
    for fn in (L.dua_sandwich_norm, L.dua_sandwich_norm_bwd):
        for kw, text in ((dict(D=0), "D must"), (dict(D=8193), "D must"), (dict(rows=-1), "D must"), (dict(dtype=3), "dtype"), (dict(param_dtype=1), "dtype"),
                         (dict(post=3), "norm kinds"), (dict(post=0, post_w=P), "off"), (dict(gate=P, gate_rows=3), "gate"), (dict(gate=P, gate_rows=0), "gate"),
                         (dict(x=None), "null"), (dict(eps=-1.0), "eps"), (dict(stats=P + 4), "stats")):
            refuses(fn, norm(**kw), text)
    refuses(L.dua_sandwich_norm, norm(z=None), "output")
    refuses(L.dua_sandwich_norm_bwd, norm(post_w=P), "gradient")
    refuses(L.dua_sandwich_norm_bwd, norm(dz=None), "null")
    refuses(L.dua_sandwich_norm_bwd, norm(), "workspace")
    assert L.dua_sandwich_norm(ctypes.byref(norm(rows=0, x=None)), None) == 0
    assert L.dua_sandwich_norm_bwd_workspace_bytes(ctypes.byref(norm(D=0))) == 0

    def att(**kw):
        a = _lib.RelAttentionArgs(q=P, k=P, v=P, B=1, Tq=4, Tk=4, heads=2, kv_heads=1, ch=32, table=P, bucket_map=P, radius=16, num_buckets=8, scale=1.0,
                                  out=P, lse=P, dout=P, dq=P, dk=P, dv=P, dtable=P)
        for n, v in kw.items():
            setattr(a, n, v)
        return a

    assert L.dua_rel_attention(None, None) == -1 and L.dua_rel_attention_bwd(None, None) == -1
    for fn in (L.dua_rel_attention, L.dua_rel_attention_bwd):
        for kw, text in ((dict(ch=0), "width"), (dict(ch=132), "width"), (dict(ch=30), "width"), (dict(ch=20, dtype=1), "width"), (dict(q_row=1 << 24), "strides"), (dict(k_row=-8), "strides"), (dict(kv_heads=3), "kv_heads"), (dict(dtype=5), "dtype"), (dict(table_dtype=2), "dtype"),
                         (dict(radius=0), "radius"), (dict(radius=1025), "radius"), (dict(num_buckets=0), "radius"), (dict(table=None), "table"),
                         (dict(bucket_map=None), "map"), (dict(k=None), "null"), (dict(q=None), "null"), (dict(Tk=1 << 29), "lengths"), (dict(Tq=-1), "lengths"),
                         (dict(B=1 << 22), "blocks")):
            refuses(fn, att(**kw), text)
    refuses(L.dua_rel_attention, att(out=None), "output")
    refuses(L.dua_rel_attention_bwd, att(dtable=None), "dtable")
    refuses(L.dua_rel_attention_bwd, att(lse=None), "null")
    refuses(L.dua_rel_attention_bwd, att(dk=None), "output")
    refuses(L.dua_rel_attention_bwd, att(), "workspace")
    assert L.dua_rel_attention(ctypes.byref(att(Tq=0, q=None)), None) == 0 and L.dua_rel_attention(ctypes.byref(att(B=0)), None) == 0

    def lp(**kw):
        a = _lib.TokenLogprobsArgs(logits=P, rows=2, V=100, ld=100, ids=P, k=5, inv_temperature=1.0, logprob=P, entropy=P, lse=P, top_ids=P, top_logprobs=P,
                                   stats=P, dlogprob=P, dtop=P, dlogits=P + 8192, ldd=100)
        for n, v in kw.items():
            setattr(a, n, v)
        return a

    assert L.dua_token_logprobs(None, None) == -1 and L.dua_token_logprobs_bwd(None, None) == -1
    for fn in (L.dua_token_logprobs, L.dua_token_logprobs_bwd):
        for kw, text in ((dict(V=0), "V in"), (dict(ld=99), "ld"), (dict(rows=-1), "rows"), (dict(rows=1 << 24), "rows"), (dict(k=65), "k must"), (dict(k=-1), "k must"),
                         (dict(V=4, k=5), "k must"), (dict(inv_temperature=0.0), "inv_temperature"), (dict(inv_temperature=math.nan), "inv_temperature"),
                         (dict(logits=None), "null"), (dict(stats=P + 4), "stats"), (dict(dtype=-1), "dtype")):
            refuses(fn, lp(**kw), text)
    refuses(L.dua_token_logprobs, lp(entropy=None), "output")
    refuses(L.dua_token_logprobs, lp(V=1 << 20, ld=1 << 20), "workspace")
    refuses(L.dua_token_logprobs_bwd, lp(ldd=99), "null operand")
    refuses(L.dua_token_logprobs_bwd, lp(ids=None), "null operand")
    refuses(L.dua_token_logprobs_bwd, lp(dtop=None), "null operand")
    refuses(L.dua_token_logprobs_bwd, lp(dlogits=P, ldd=128), "in place")
    assert L.dua_token_logprobs(ctypes.byref(lp(rows=0, logits=None)), None) == 0


def test_rel_attention_block_count():
    """B * heads * blocks of 64 rows stay below 2^23 whatever the factors (their product may pass 2^64), and the forward pass counts queries alone: a
    long cache is no reason to refuse a decoding step."""
    from diffusion_uncertainty_amd import _lib
    L = _lib.lib()
    P = 4096
    att = lambda **kw: _lib.RelAttentionArgs(**{**dict(q=P, k=P, v=P, B=1, Tq=4, Tk=4, heads=2, kv_heads=1, ch=32, table=P, bucket_map=P, radius=16, num_buckets=8,
                                                       scale=1.0, out=P, lse=P, dout=P, dq=P, dk=P, dv=P, dtable=P), **kw})
    T = (1 << 25) - 64
    for kw in (dict(B=1 << 30, heads=1 << 15, kv_heads=1 << 15, Tq=T, Tk=T), dict(B=1 << 23), dict(B=(1 << 31) - 1, heads=65535, kv_heads=1)):
        for fn in (L.dua_rel_attention, L.dua_rel_attention_bwd):
            assert fn(ctypes.byref(att(**kw)), None) == -1 and "blocks" in L.dua_last_error().decode(), L.dua_last_error()
        assert L.dua_rel_attention_workspace_bytes(ctypes.byref(att(**kw)), 0) == 0
    cache = att(B=8, Tq=1, Tk=600000, heads=128, kv_heads=8, ch=128, dtype=1)
    assert L.dua_rel_attention_workspace_bytes(ctypes.byref(cache), 0) > 0                       # split keys
    assert L.dua_rel_attention_workspace_bytes(ctypes.byref(cache), 1) == 0
    assert L.dua_rel_attention_bwd(ctypes.byref(cache), None) == -1 and "blocks" in L.dua_last_error().decode()


def test_rel_attention_shares_of_the_queries_fill_the_chip_once():
    """Backward, one query head a kv head: a share of the queries costs fp32 sums of dk and dv in the workspace.  Sixteen-bit types take as many whole shares as
    512 workgroups have room for (none at 320), fp32 one more where that leaves places empty."""
    from diffusion_uncertainty_amd import _lib
    L = _lib.lib()
    P = 4096

    def shares(dtype, B, T=1024, H=8, ch=64):
        a = _lib.RelAttentionArgs(q=P, k=P, v=P, dtype=dtype, B=B, Tq=T, Tk=T, heads=H, kv_heads=H, ch=ch, table=P, table_dtype=dtype, bucket_map=P, radius=1,
                                  num_buckets=2, scale=1.0, out=P, lse=P, dout=P, dq=P, dk=P, dv=P, dtable=P)
        n = L.dua_rel_attention_workspace_bytes(ctypes.byref(a), 1)
        one = 2 * B * T * H * ch * 4                                                 # dk and dv of a share
        return n // one

    assert [shares(1, B) for B in (1, 2, 3, 4, 5, 6, 7, 8)] == [8, 4, 2, 2, 0, 0, 0, 0]
    assert [shares(2, B) for B in (3, 5)] == [2, 0]
    assert [shares(0, B) for B in (1, 2, 3, 4)] == [4, 2, 2, 0]


def test_rel_attention_splits_keys_where_the_chip_is_empty():
    """Forward, tiles of queries: the number of shares of the keys by the workspace they take (ch sums, a maximum and a sum a row and share)."""
    from diffusion_uncertainty_amd import _lib
    L = _lib.lib()
    P = 4096

    def shares(dtype, B, Tq, Tk, H=8, ch=64):
        a = _lib.RelAttentionArgs(q=P, k=P, v=P, dtype=dtype, B=B, Tq=Tq, Tk=Tk, heads=H, kv_heads=H, ch=ch, table=P, table_dtype=dtype, bucket_map=P, radius=1,
                                  num_buckets=2, scale=1.0, out=P)
        n = L.dua_rel_attention_workspace_bytes(ctypes.byref(a), 0)
        one = B * H * Tq * (ch + 2) * 4
        assert n % one == 0
        return n // one                                                              # 0: none

    assert [shares(1, 1, 128, 2000), shares(1, 1, 1024, 1024), shares(1, 1, 1024, 4096)] == [7, 4, 8]
    assert [shares(1, 2, 1024, 1024), shares(2, 3, 1024, 1024), shares(1, 3, 1024, 2048)] == [0, 0, 0]
    assert [shares(1, 2, 1024, 4096), shares(2, 3, 1024, 4096), shares(1, 4, 1024, 4096)] == [4, 2, 0]
    assert [shares(0, 1, 1024, 1024), shares(0, 1, 1920, 2048), shares(0, 2, 1024, 1024)] == [4, 3, 0]


def test_token_logprobs_parts_have_no_cliff():
    """Long rows are dealt in parts up to 512 of them, short ones below 256: the number of parts by the workspace (4 sums and k pairs each)."""
    from diffusion_uncertainty_amd import _lib
    L = _lib.lib()

    def parts(rows, V, dtype, k=5):
        a = _lib.TokenLogprobsArgs(rows=rows, V=V, ld=V, k=k, dtype=dtype, inv_temperature=1.0)
        return L.dua_token_logprobs_workspace_bytes(ctypes.byref(a)) // (rows * (4 + 2 * k) * 4)

    assert [parts(r, 128000, 1) for r in (4, 255, 256, 384, 512, 513)] == [31, 3, 4, 3, 2, 0]
    assert [parts(r, 65536, 0) for r in (255, 256, 512)] == [3, 4, 2]
    assert [parts(r, 65536, 2) for r in (255, 256, 512)] == [3, 0, 0]
    assert parts(4, 8191, 0) == 0 and parts(4, 8192, 0) == 2


def test_token_logprobs_refuses_a_temperature_without_log2_units():
    from diffusion_uncertainty_amd import _lib
    L = _lib.lib()
    P = 4096
    for t, ok in ((3e38, False), (2.4e38, False), (1e38, True)):
        a = _lib.TokenLogprobsArgs(logits=P, rows=0, V=100, ld=100, k=0, inv_temperature=t, logprob=P, entropy=P, lse=P, stats=P)
        assert (L.dua_token_logprobs(ctypes.byref(a), None) == 0) == ok
        assert ok or "inv_temperature" in L.dua_last_error().decode()
