"""Token operators on the HIP library (attention with a bucketed relative bias, sandwich norm, token log probabilities) against
oracle/tokens.py in 64 bits, at the sizes, masks, strides and alignments where they can go wrong.

Tolerances count roundings.  u = 2^-24 is half a step of fp32, e = finfo(dtype).eps / 2 of the tensors' type.  A sum of n terms added in chains
and trees of depth d is off by at most d u times the sum of the terms' magnitudes; the oracle returns those magnitudes."""
import math

import pytest
import torch

from oracle import tokens as oracle

pytestmark = pytest.mark.gpu
dev = "cuda"
U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def half_step(dt):
    return torch.finfo(dt).eps / 2


def close(got, want, tol, what=""):
    """|got - want| <= tol elementwise.  An fp16 result below 2^-14 is rounded to a multiple of 2^-24, off by up to 2^-25 whatever its size
    (3.2636e-05 becomes 3.2663e-05: 2.7e-08 off, 1.7 times 2^-11 of the value): that half step is added for fp16."""
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -25
    got, want = got.detach().cpu().to(torch.float64), want.detach().to(torch.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    same = (got == want) | (got.isnan() & want.isnan())
    err = torch.where(same, 0.0, (got - want).abs())
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / tol).nan_to_num(nan=1e30).max()):.3g} x the bound"


def rnd(g, *s, dtype=torch.float32, scale=1.0):
    return (torch.randn(*s, generator=g) * scale).to(dtype)


# ------------------------------------------------------------------------------------------------------------- attention
def attention_bounds(r, dt, ch, Tk, Tq, rep):
    """A logit is a chain of ch products, the scale, the bias, the base change: its error is at most (ch + 8) u times its magnitude `logit`; with the
    exponential and its argument's rounding a probability before normalising is off by the factor 1 +- dl (both it and the sum: 2 dl, plus
    the sum's chain).  P is rounded to the tensors' type before P v, dS before dS k / dS^T q; sums over keys are chains of Tk."""
    e = half_step(dt)
    ep = 0.0 if dt == torch.float32 else e
    dl = ((ch + 8) * r["logit"] + 8) * U                                            # [B, H, Tq]
    dp = 2 * dl + (Tk + 8) * U
    rows = lambda t: t.permute(0, 2, 1).repeat_interleave(ch, 2)                      # [B, H, Tq] -> [B, Tq, H ch]
    sub = 2.0 ** -25 * max(Tk, rep * Tq) * 6.0 if dt == torch.float16 else 0.0       # fp16: half a subnormal step of P / dS times |operand| <= 6
    tol = dict(out=r["pv"] * (rows(dp) + ep + Tk * U) + e * r["out"].abs() + sub,
               lse=dp + 4 * U * r["lse"].abs().nan_to_num(posinf=0.0) + 1e-30)
    if "dq" in r:
        w = dp.max()
        # dS: P's factor, dP's chain over ch, D's chain (from the output and what its rounding left: e^2), its own rounding
        ds = w + (ch + 4) * U + e * e + ep
        tol.update(dq=r["adq"] * (ds + (Tk + 8) * U) + e * r["dq"].abs() + sub, dk=r["adk"] * (ds + (rep * Tq + 8) * U) + e * r["dk"].abs() + sub,
                   dv=r["adv"] * (w + ep + (rep * Tq + 8) * U) + e * r["dv"].abs() + sub,
                   dtable=r["adtable"] * (ds + (600 + Tq + Tk) * U) + e * r["dtable"].abs())
    return tol


def attention_case(dt, B, Tq, Tk, H, Hk, ch, causal=False, klen=None, qstart=None, radius=16, nb=8, seed=0, grads=True, bi=None, table_dt=None,
                   scale=None):
    from diffusion_uncertainty_amd import ops
    g = torch.Generator().manual_seed(seed)
    q, k, v = rnd(g, B, Tq, H * ch, dtype=dt), rnd(g, B, Tk, Hk * ch, dtype=dt), rnd(g, B, Tk, Hk * ch, dtype=dt)
    do, table = rnd(g, B, Tq, H * ch, dtype=dt), rnd(g, nb, H, dtype=table_dt or dt)
    bk = ops.RelativeBuckets(nb, radius, (not causal) if bi is None else bi, device=dev)
    kl = None if klen is None else torch.tensor(klen, dtype=torch.int32)
    qs = None if qstart is None else torch.tensor(qstart, dtype=torch.int32)
    r = oracle.rel_attention(q, k, v, table, bk.map.cpu(), H, Hk, causal, scale, kl, qs, do if grads else None)
    D = lambda t: None if t is None else t.to(dev)
    kw = dict(heads=H, kv_heads=Hk, causal=causal, scale=scale, klen=D(kl), qstart=D(qs))
    kg, vg = D(k), D(v)
    if klen is not None:                                                            # what lies behind klen must not matter
        for b, n in enumerate(klen):
            kg[b, max(n, 0):] = math.nan
            vg[b, max(n, 0):] = math.inf
    tol = attention_bounds(r, dt, ch, max(Tk, 1), Tq, H // Hk)
    args = (D(q), kg, vg, D(table), bk)
    out, lse = ops.rel_attention(*args, want_lse=True, **kw)
    close(out, r["out"], tol["out"], "out")
    close(lse.lse, r["lse"], tol["lse"], "lse")
    if grads:
        got = ops.rel_attention_bwd(*args, out, lse, D(do), **kw)
        for n, t in zip(("dq", "dk", "dv", "dtable"), got):
            close(t, r[n], tol[n] + 1e-30, n)
        again = ops.rel_attention_bwd(*args, out, lse, D(do), **kw)
        for a, b in zip(got, again):
            assert torch.equal(a, b), "two runs differ"
    return out


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("B,Tq,Tk,H,Hk,ch,causal", [(2, 1, 1, 1, 1, 64, False), (1, 65, 65, 2, 2, 64, True), (2, 129, 129, 4, 2, 72, False),
                                                    (1, 200, 200, 4, 1, 128, True), (3, 7, 130, 2, 1, 32, False), (1, 66, 66, 2, 2, 96, True)])
def test_rel_attention_and_gradients(dt, B, Tq, Tk, H, Hk, ch, causal):
    attention_case(dt, B, Tq, Tk, H, Hk, ch, causal)


@pytest.mark.parametrize("dt", DTYPES)
def test_rel_attention_lengths_offsets_and_empty_rows(dt):
    # padded batch with an empty sequence, garbage behind klen; offsets in front of, inside and past the keys
    attention_case(dt, 4, 70, 90, 2, 1, 40, False, klen=[90, 1, 0, 63], seed=1)
    attention_case(dt, 4, 70, 90, 2, 1, 40, True, klen=[90, 40, 90, 0], qstart=[20, 0, -30, 5], seed=2)
    attention_case(dt, 3, 9, 300, 2, 2, 64, True, klen=[300, 130, 300], qstart=[291, 121, 2000], seed=3, radius=64, nb=16)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("Tk,ch,H,Hk", [(1, 64, 2, 2), (257, 64, 4, 2), (1000, 128, 2, 1), (4100, 72, 1, 1), (130, 24, 3, 3), (63, 40, 34, 2)])
def test_rel_attention_decoding(dt, Tk, ch, H, Hk):
    n = [Tk, max(Tk // 2, 1), 0]
    attention_case(dt, 3, 1, Tk, H, Hk, ch, True, klen=n, qstart=[max(x - 1, 0) for x in n], seed=Tk, grads=False)
    attention_case(dt, 3, 1, Tk, H, Hk, ch, False, klen=n, qstart=[5, 0, 3], seed=Tk, grads=False)


@pytest.mark.parametrize("ch", [8, 24, 40, 56, 88, 104, 120])
def test_rel_attention_head_widths(ch):
    for dt in DTYPES:
        attention_case(dt, 1, 37, 67, 2, 1, ch, False, seed=ch)
    for w in (ch - 4, ch + 4):
        attention_case(torch.float32, 1, 37, 67, 2, 1, w, False, seed=w)


@pytest.mark.parametrize("dt", DTYPES)
def test_rel_attention_few_queries_and_split_keys(dt):
    """Several tokens a step in the 16 columns of a tile, shared kv heads; tiles of queries whose keys are split over workgroups; their gradients."""
    for B, Tq, Tk, H, Hk, ch in [(2, 5, 700, 4, 2, 64), (1, 16, 300, 1, 1, 72), (3, 2, 33, 8, 1, 128), (1, 40, 1500, 2, 1, 64), (2, 17, 1030, 1, 1, 128)]:
        n = [Tk, Tk // 2, Tk - 3][:B]
        attention_case(dt, B, Tq, Tk, H, Hk, ch, True, klen=n, qstart=[x - Tq for x in n], seed=Tq)
        attention_case(dt, B, Tq, Tk, H, Hk, ch, False, klen=n, qstart=[x - Tq for x in n], seed=Tq + 1, grads=Tq < 17)


@pytest.mark.parametrize("dt", DTYPES)
def test_rel_attention_unwritten_slots_behind_the_last_query(dt):
    """A cache without klen whose slots behind the last causal query hold anything: not read, by either pass."""
    from diffusion_uncertainty_amd import ops
    g = torch.Generator().manual_seed(2)
    for Tq, qs in ((1, 40), (3, 70), (50, 31)):
        B, Tk, H, ch = 2, 128, 2, 64
        q, k, v, do = rnd(g, B, Tq, H * ch, dtype=dt), rnd(g, B, Tk, H * ch, dtype=dt), rnd(g, B, Tk, H * ch, dtype=dt), rnd(g, B, Tq, H * ch, dtype=dt)
        table, bk = rnd(g, 8, H, dtype=dt).to(dev), ops.RelativeBuckets(8, 16, False, device=dev)
        qst = torch.full((B,), qs, dtype=torch.int32, device=dev)
        kw = dict(heads=H, causal=True, qstart=qst)
        res = []
        for fill in (0.0, math.nan):
            kk, vv = k.to(dev), v.to(dev)
            kk[:, qs + Tq:], vv[:, qs + Tq:] = fill, fill
            out, s = ops.rel_attention(q.to(dev), kk, vv, table, bk, want_lse=True, **kw)
            res.append((out, *ops.rel_attention_bwd(q.to(dev), kk, vv, table, bk, out, s, do.to(dev), **kw)))
        for a, b in zip(*res):
            assert torch.isfinite(a).all() and torch.equal(a, b)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Tq,Tk,H,Hk,ch", [(1, 1000, 4, 4, 64), (1, 3000, 16, 2, 128), (4, 333, 4, 1, 72), (2, 90, 2, 1, 40)])
def test_rel_attention_few_queries_are_off_by_their_own_rounding(dt, Tq, Tk, H, Hk, ch):
    """Decoding: P is not rounded to the tensors' type but to two numbers of it (e^2; fp16: half a subnormal step of the second, beside a largest P of at least
    1), so nothing of e is left but the output's own rounding."""
    from diffusion_uncertainty_amd import ops
    g = torch.Generator().manual_seed(19)
    e = half_step(dt)
    q, k, v = rnd(g, 3, Tq, H * ch, dtype=dt), rnd(g, 3, Tk, Hk * ch, dtype=dt), rnd(g, 3, Tk, Hk * ch, dtype=dt)
    table, bk = rnd(g, 8, H, dtype=dt), ops.RelativeBuckets(8, 16, True, device=dev)
    n = torch.tensor([Tk, Tk - 7, Tk // 2], dtype=torch.int32)
    r = oracle.rel_attention(q, k, v, table, bk.map.cpu(), H, Hk, True, None, n, n - Tq)
    out = ops.rel_attention(q.to(dev), k.to(dev), v.to(dev), table.to(dev), bk, heads=H, kv_heads=Hk, causal=True, klen=n.to(dev), qstart=(n - Tq).to(dev))
    dp = 2 * ((ch + 8) * r["logit"] + 8) * U + (Tk + 8) * U
    rows = dp.permute(0, 2, 1).repeat_interleave(ch, 2)
    sub = 2.0 ** -25 * Tk * v.abs().max().double() if dt == torch.float16 else 0.0
    close(out, r["out"], r["pv"] * (rows + e * e + Tk * U) + e * r["out"].abs() + sub, "out")


def test_rel_attention_table_of_the_lowest_value():
    from diffusion_uncertainty_amd import ops
    g = torch.Generator().manual_seed(4)
    q, k, v, do = (rnd(g, 1, 30, 64).to(dev) for _ in range(4))
    bk = ops.RelativeBuckets(8, 16, True, device=dev)
    t1, t2 = rnd(g, 8, 2).to(dev), None
    t1[5] = torch.finfo(torch.float32).min
    t2 = t1.clone()
    t2[5] = -math.inf
    for a, b in zip(*[(o, *ops.rel_attention_bwd(q, k, v, t, bk, o, s, do, heads=2)) for t in (t1, t2) for o, s in [ops.rel_attention(q, k, v, t, bk, heads=2, want_lse=True)]]):
        assert torch.isfinite(a).all() and torch.equal(a, b)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("mask", [-65504.0, -1e6, -1e9, -9e29, 1e9])
def test_rel_attention_masks_of_large_finite_values(dt, mask):
    """A bias of +-1e9: a query that sees nothing else has the softmax of its scores alone (a common shift), queries that see other keys too do not see
    those of -1e9.  Beside 65504 a score is rounded to half a step of 65504 log2 e, 2^-8 log2 units; so are the row's maximum with its sum, and lse (2^-9
    and once more 2^-8 on its way back): P is off by 3 2^-8 ln 2 + 2^-9 = 0.011 at most, before normalising and after."""
    from diffusion_uncertainty_amd import ops
    g = torch.Generator().manual_seed(41)
    x = 2 * 0.011
    bk = ops.RelativeBuckets(8, 16, True, device=dev)
    far = int(bk.map[0])                                                             # the bucket of keys 16 and more to the left
    for B, Tq, Tk, H, Hk, ch in ((2, 70, 100, 2, 1, 64), (1, 1, 100, 4, 2, 64), (1, 2, 1000, 2, 2, 40), (1, 40, 900, 1, 1, 128)):
        q, k, v, do = rnd(g, B, Tq, H * ch, dtype=dt), rnd(g, B, Tk, Hk * ch, dtype=dt), rnd(g, B, Tk, Hk * ch, dtype=dt), rnd(g, B, Tq, H * ch, dtype=dt)
        table = rnd(g, 8, H)
        table[far] = mask
        D = lambda t: t.to(dev)
        for start, causal in ((5000, False), (5000, True), (Tk - Tq, True), (Tk // 2, False)):
            alone = start == 5000
            qs = torch.full((B,), start, dtype=torch.int32)
            t0 = table.clone()
            if alone:
                t0[far] = 0.0
            elif mask > 0:
                continue
            r = oracle.rel_attention(q, k, v, t0, bk.map.cpu(), H, Hk, causal, None, None, qs, do)
            tol = attention_bounds(r, dt, ch, Tk, Tq, H // Hk)
            kw = dict(heads=H, kv_heads=Hk, causal=causal, qstart=D(qs))
            out, s = ops.rel_attention(D(q), D(k), D(v), D(table), bk, want_lse=True, **kw)
            got = ops.rel_attention_bwd(D(q), D(k), D(v), D(table), bk, out, s, D(do), **kw)
            y = x if alone else 0.0
            close(out, r["out"], tol["out"] + y * r["pv"], "out")
            for n, t in zip(("dq", "dk", "dv", "dtable"), got):
                close(t, r[n], tol[n] + y * r["a" + n] + 1e-30, n)


def test_rel_attention_table_without_a_value():
    """+inf and NaN in the table are not clipped: a query that sees them has no result."""
    from diffusion_uncertainty_amd import ops
    g = torch.Generator().manual_seed(42)
    q, k, v = (rnd(g, 1, 40, 64).to(dev) for _ in range(3))
    bk = ops.RelativeBuckets(8, 16, True, device=dev)
    near = min(d for d in range(17) if bk.map[16 - d] == bk.map[0])                  # the bucket's nearest distance
    for bad in (math.inf, math.nan):
        table = rnd(g, 8, 2)
        table[int(bk.map[0]), 1] = bad
        for n in (1, 40):
            out = ops.rel_attention(q[:, :n], k, v, table.to(dev), bk, heads=2, qstart=torch.full((1,), 39 if n == 1 else 0, dtype=torch.int32, device=dev)).view(n, 2, 32)
            sees = torch.arange(40 - n, 40) >= near
            assert torch.isfinite(out[:, 0]).all() and out[:, 1].isnan().all(1).cpu().tolist() == sees.tolist()


def test_rel_attention_table_types_scale_and_wide_radius():
    attention_case(torch.bfloat16, 1, 80, 80, 2, 2, 64, True, table_dt=torch.float32, scale=0.3)
    attention_case(torch.float32, 1, 40, 1300, 1, 1, 16, False, radius=1024, nb=64, seed=4)
    attention_case(torch.float32, 1, 70, 200, 1, 1, 128, False, radius=1024, nb=64, seed=7)
    attention_case(torch.float16, 1, 300, 300, 1, 1, 16, False, radius=3, nb=4, seed=5)
    attention_case(torch.float32, 1, 50, 50, 1, 1, 32, True, bi=True, seed=6)


def test_rel_attention_custom_map_and_minus_infinite_bias():
    """Entries outside the table add nothing; a bucket of -inf masks its distances, a query with nothing else left is empty."""
    from diffusion_uncertainty_amd import ops
    g = torch.Generator().manual_seed(3)
    B, T, H, ch = 1, 40, 2, 32
    q, k, v, do = (rnd(g, B, T, H * ch) for _ in range(4))
    m = torch.tensor([0, 1, -1, 2, 7, 1, 0], dtype=torch.int32)
    table = rnd(g, 3, H)
    table[0] = -math.inf                                                             # everything at distance >= 3
    table[1, 1] = -math.inf
    r = oracle.rel_attention(q, k, v, table, m, H, H, True, None, None, None, do)
    bk = ops.RelativeBuckets.from_map(m.to(dev), 3)
    a = (q.to(dev), k.to(dev), v.to(dev), table.to(dev), bk)
    out, lse = ops.rel_attention(*a, heads=H, causal=True, want_lse=True)
    got = ops.rel_attention_bwd(*a, out, lse, do.to(dev), heads=H, causal=True)
    r["logit"] = r["logit"].nan_to_num(posinf=50.0).clamp(max=50.0)
    tol = attention_bounds(r, torch.float32, ch, T, T, 1)
    close(out, r["out"], tol["out"], "out")
    close(lse.lse, r["lse"], tol["lse"], "lse")
    for n, t in zip(("dq", "dk", "dv", "dtable"), got):
        close(t, r[n], tol[n] + 1e-30, n)
    # the only distance left is masked: every query is empty
    table[2] = -math.inf
    m2 = torch.zeros(3, dtype=torch.int32)
    out, lse = ops.rel_attention(*a[:3], table.to(dev), ops.RelativeBuckets.from_map(m2.to(dev), 3), heads=H, want_lse=True)
    assert (out == 0).all() and (lse.lse == -math.inf).all()


@pytest.mark.parametrize("dt", DTYPES)
def test_rel_attention_table_gradient_of_many_sequences(dt):
    """18 sequences of three or five blocks of keys: the table's gradient is added up in two launches instead of one."""
    attention_case(dt, 18, 40, 260, 2, 1, 16, radius=40, klen=[260 - 7 * b for b in range(18)], qstart=[11 * b for b in range(18)], seed=14)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("Tq,Tk,H,Hk,ch,causal,klen,qstart", [(520, 150, 2, 2, 64, False, None, None), (333, 333, 4, 2, 16, True, [300], None),
                                                              (300, 140, 1, 1, 128, True, [130], [-100]), (400, 3, 2, 1, 72, False, [0], None)])
def test_rel_attention_gradients_of_one_sequence(dt, Tq, Tk, H, Hk, ch, causal, klen, qstart):
    """Few blocks of keys: dk and dv summed over shares of the queries, some of which see none of a block's keys."""
    attention_case(dt, 1, Tq, Tk, H, Hk, ch, causal, klen=klen, qstart=qstart, seed=15)


@pytest.mark.parametrize("dt", DTYPES)
def test_rel_attention_strided_views(dt):
    """Thirds of a qkv projection, slots of a larger cache, rows that are not 16-byte aligned: the same bits as from contiguous copies."""
    from diffusion_uncertainty_amd import ops
    g = torch.Generator().manual_seed(8)
    B, T, H, ch = 2, 75, 2, 64
    C = H * ch
    bk = ops.RelativeBuckets(8, 16, True, device=dev)
    table = rnd(g, 8, H, dtype=dt).to(dev)
    for width in (3 * C, 3 * C + 1):
        qkv = rnd(g, B, T, width, dtype=dt).to(dev)
        q, k, v = qkv[..., :C], qkv[..., C:2 * C], qkv[..., 2 * C:3 * C]
        do = rnd(g, T, B, C, dtype=dt).to(dev).transpose(0, 1)
        want, lse = ops.rel_attention(q.contiguous(), k.contiguous(), v.contiguous(), table, bk, heads=H, want_lse=True)
        got, lse2 = ops.rel_attention(q, k, v, table, bk, heads=H, want_lse=True)
        assert torch.equal(got, want) and torch.equal(lse.lse, lse2.lse)
        a = ops.rel_attention_bwd(q, k, v, table, bk, got, lse, do, heads=H)
        b = ops.rel_attention_bwd(q.contiguous(), k.contiguous(), v.contiguous(), table, bk, want, lse, do.contiguous(), heads=H)
        for x, y in zip(a, b):
            assert torch.equal(x, y)
    one = rnd(g, 1, T, C, dtype=dt).to(dev)                                          # keys shared by a batch: stride 0
    q = rnd(g, B, T, C, dtype=dt).to(dev)
    assert torch.equal(ops.rel_attention(q, one.expand(B, T, C), one.expand(B, T, C), table, bk, heads=H),
                       ops.rel_attention(q, one.repeat(B, 1, 1), one.repeat(B, 1, 1), table, bk, heads=H))


def test_rel_attention_empty_tensors():
    from diffusion_uncertainty_amd import ops
    bk = ops.RelativeBuckets(8, 16, True, device=dev)
    table = torch.ones(8, 2, device=dev)
    z = lambda *s: torch.zeros(*s, device=dev)
    out, lse = ops.rel_attention(z(2, 5, 64) + 1, z(2, 0, 64), z(2, 0, 64), table, bk, heads=2, want_lse=True)
    assert (out == 0).all() and (lse.lse == -math.inf).all()
    dq, dk, dv, dt = ops.rel_attention_bwd(z(2, 5, 64) + 1, z(2, 0, 64), z(2, 0, 64), table, bk, out, lse, z(2, 5, 64) + 1, heads=2)
    assert (dq == 0).all() and dk.shape == (2, 0, 64) and (dt == 0).all()
    out, lse = ops.rel_attention(z(2, 0, 64), z(2, 5, 64), z(2, 5, 64), table, bk, heads=2, want_lse=True)
    dq, dk, dv, dt = ops.rel_attention_bwd(z(2, 0, 64), z(2, 5, 64), z(2, 5, 64), table, bk, out, lse, z(2, 0, 64), heads=2)
    assert out.shape == (2, 0, 64) and (dk == 0).all() and (dv == 0).all() and (dt == 0).all()
    out, lse = ops.rel_attention(z(0, 5, 64), z(0, 5, 64), z(0, 5, 64), table, bk, heads=2, want_lse=True)
    assert out.shape == (0, 5, 64)
    assert (ops.rel_attention_bwd(z(0, 5, 64), z(0, 5, 64), z(0, 5, 64), table, bk, out, lse, out, heads=2)[3] == 0).all()


def test_rel_attention_gradient_against_differences():
    """Central differences of the 64-bit definition along random directions against the kernels' gradients in fp32."""
    from diffusion_uncertainty_amd import ops
    g = torch.Generator().manual_seed(21)
    B, T, H, Hk, ch = 2, 33, 4, 2, 16
    bk = ops.RelativeBuckets(8, 16, False, device=dev)
    x = dict(q=rnd(g, B, T, H * ch), k=rnd(g, B, T, Hk * ch), v=rnd(g, B, T, Hk * ch), table=rnd(g, 8, H))
    do, kl = rnd(g, B, T, H * ch), torch.tensor([33, 20], dtype=torch.int32)
    f = lambda d: (oracle.rel_attention(d["q"], d["k"], d["v"], d["table"], bk.map.cpu(), H, Hk, True, klen=kl)["out"] * do.double()).sum().item()
    a = [x[n].to(dev) for n in x] + [bk]
    kw = dict(heads=H, kv_heads=Hk, causal=True, klen=kl.to(dev))
    out, lse = ops.rel_attention(*a, want_lse=True, **kw)
    grads = dict(zip(x, ops.rel_attention_bwd(*a, out, lse, do.to(dev), **kw)))
    h = 1e-4
    for n in x:
        d = torch.randn(x[n].shape, generator=g, dtype=torch.float64)
        diff = (f({**x, n: x[n].double() + h * d}) - f({**x, n: x[n].double() - h * d})) / (2 * h)
        have = (grads[n].cpu().double() * d).sum().item()
        size = (grads[n].cpu().double() * d).abs().sum().item()
        assert abs(diff - have) < 1e-5 * size + 1e-6, (n, diff, have)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("B,Hk", [(2, 4), (13, 5)])
def test_rel_attention_kv_heads_on_eight_dies(dt, B, Hk):
    """8 and 65 kv heads: their blocks are dealt to the eight XCDs, the last round of 65 partly filled."""
    attention_case(dt, B, 40, 70, 2 * Hk, Hk, 16, True, qstart=[30 - b for b in range(B)], seed=16)


@pytest.mark.parametrize("dt", DTYPES)
def test_rel_attention_joins_of_more_than_64_splits(dt):
    """One head over 20000 keys: 128 splits (one query), 78 (a tile of queries); two wavefronts hold the splits' weights."""
    attention_case(dt, 1, 1, 20000, 1, 1, 16, True, klen=[19990], qstart=[19989], seed=17, grads=False)
    attention_case(dt, 1, 40, 20000, 1, 1, 16, False, klen=[19990], qstart=[10000], seed=18)


FORMS = [(70, 150), (3, 100), (1, 3000), (40, 1500)]                   # tiles of queries, few queries, and both with split keys


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Tq,Tk", FORMS)
def test_rel_attention_keeps_what_the_outputs_rounding_left(dt, Tq, Tk):
    """Equal keys and no bias: every P is 1 and rounds to itself, so out + out_lo is the mean of the values (3 + a normal number) but for fp32's roundings -
    a logit's in P and in their sum, 32 in an instruction and one for every 16 keys in the sums - and out_lo's own (e^2; fp16: half a subnormal step)."""
    from diffusion_uncertainty_amd import ops
    g = torch.Generator().manual_seed(51)
    H, ch, e = 2, 64, half_step(dt)
    q, v = rnd(g, 1, Tq, H * ch, dtype=dt, scale=0.1), (3.0 + rnd(g, 1, Tk, H * ch)).to(dt)
    k = rnd(g, 1, 1, H * ch, dtype=dt).repeat(1, Tk, 1)
    bk = ops.RelativeBuckets(8, 16, True, device=dev)
    out, s = ops.rel_attention(q.to(dev), k.to(dev), v.to(dev), torch.zeros(8, H, device=dev), bk, heads=H, want_lse=True)
    r = oracle.rel_attention(q, k, v, torch.zeros(8, H), bk.map.cpu(), H, H)
    tol = r["pv"] * 2 * ((ch + 8) * r["logit"].max() + 8 + 40 + Tk / 16) * U + e * e * r["out"].abs() + (2.0 ** -25 if dt == torch.float16 else 0.0)
    lo = s.out_lo.permute(0, 2, 1, 3).reshape(1, Tq, H * ch)
    close(out.double() + lo.double(), r["out"], tol, "out + out_lo")
    bare = (r["out"].to(dt).double() - r["out"]).abs()
    assert (bare > 4 * tol).any(), "the bound would not tell out from out + out_lo"


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Tq,Tk", FORMS)
def test_rel_attention_gradients_of_decided_queries(dt, Tq, Tk):
    """Queries that all find two equal keys whose values are a step or two of their type apart: the output lies between two numbers, dS = P (dP - D) is the
    small difference of large terms, and D = dO . o has to be better than the rounded output.

    Bounds, one query: dS is off by its own rounding e |dS| and by P times (dP's and D's chains of ch products, (ch + 4) u each of |dO| . |v| and |dO| . |o|;
    what out_lo's rounding leaves of D, e^2 |dO| . |o| and in fp16 2^-25 |dO|; the forward's rounding of the other keys' P, e |dO| . sum P |v|; P's own
    relative error w times |dP - D|).  dk and the table take D corrected by the row's sum of dS: what is left of the output's errors drops out, with
    out_lo or without; the table takes dS unrounded."""
    from diffusion_uncertainty_amd import ops
    g = torch.Generator().manual_seed(52)
    H, ch, e, F = 8, 16, half_step(dt), torch.float64
    q, k = rnd(g, 1, Tq, H, ch, scale=0.3), rnd(g, 1, Tk, H, ch, scale=0.3)
    best = Tk // 3
    q[..., 0], k[..., 0], k[:, best, :, 0] = 8.0, 0.0, 8.0
    k[:, best + 1] = k[:, best]
    v, do = rnd(g, 1, Tk, H * ch, dtype=dt), rnd(g, 1, Tq, H * ch, dtype=dt)
    v[:, best + 1] = (v[:, best].float() * (1 + 2 * e)).to(dt)
    q, k = q.to(dt).view(1, Tq, H * ch), k.to(dt).view(1, Tk, H * ch)
    m = ops.RelativeBuckets(8, 16, True, device="cpu").map
    qs, scale = Tk // 2, 0.25
    cell = m.long()[(torch.arange(Tk)[None] - (torch.arange(Tq)[:, None] + qs)).clamp(-16, 16) + 16].reshape(-1)
    table = lambda t: torch.zeros(8, dtype=F).index_add_(0, cell, t.reshape(-1))
    want, tol, seen = {n: [] for n in ("dq", "dk", "dtable")}, {n: [] for n in ("dq", "dk", "dtable")}, []
    for h in range(H):
        Q, K, V, G = (t[0].view(-1, H, ch)[:, h].to(F) for t in (q, k, v, do))
        P = torch.softmax(scale * Q @ K.T, 1)
        others = P * ((torch.arange(Tk) != best) & (torch.arange(Tk) != best + 1))
        assert others.sum(1).max() < 2.0 ** -8                                        # (the two keys' own P are 1 before they are normalised)
        O, dP = P @ V, G @ V.T
        dP_D = dP - (G * O).sum(1, keepdim=True)
        dS = P * dP_D
        w = 2 * ((ch + 8) * (scale * Q.abs() @ K.abs().T * (P > 1e-12)).max() + 8) * U + (Tk + 8) * U
        GO = (G.abs() * O.abs()).sum(1, keepdim=True)
        chains = (ch + 4) * U * (G.abs() @ V.abs().T + GO) + w * dP_D.abs()
        rest = e * e * GO + (2.0 ** -25 if dt == torch.float16 else 0.0) * G.abs().sum(1, keepdim=True) + e * (G.abs() * (others @ V.abs())).sum(1, keepdim=True)
        far = 2.0 ** -32 * dS.abs().max() if dt == torch.float16 else 0.0              # fp16 operands far below their column's largest
        err_q, err_k = e * dS.abs() + P * (chains + rest) + far, e * dS.abs() + P * chains + far
        want["dq"].append(scale * dS @ K)
        want["dk"].append(scale * dS.T @ Q)
        want["dtable"].append(table(dS))
        tol["dq"].append(e * want["dq"][h].abs() + scale * (err_q + (Tk + 8) * U * dS.abs()) @ K.abs())
        tol["dk"].append(e * want["dk"][h].abs() + scale * (err_k + (Tq + 8) * U * dS.abs()).T @ Q.abs())
        tol["dtable"].append(U * want["dtable"][h].abs() + table(P * chains + (600 + Tq + Tk) * U * dS.abs()) + 1e-30)
        # what a D of the rounded output alone would do to dq and, uncorrected, to the table
        off = (G * (O.to(dt).to(F) - O)).sum(1, keepdim=True)
        seen.append([bool((scale * off * (P @ K)).abs().gt(4 * tol["dq"][h]).any()), bool(table(off * P).abs().gt(4 * tol["dtable"][h]).any())])
        if dt == torch.float16:
            tol["dq"][h], tol["dk"][h] = tol["dq"][h] + 2.0 ** -25, tol["dk"][h] + 2.0 ** -25
    assert all(any(x) for x in zip(*seen)), "the bounds would not tell"
    want, tol = ({n: torch.stack(t, -1 if n == "dtable" else 1) for n, t in d.items()} for d in (want, tol))
    bk = ops.RelativeBuckets.from_map(m.to(dev), 8)
    kw = dict(heads=H, scale=scale, qstart=torch.full((1,), qs, dtype=torch.int32, device=dev))
    a = (q.to(dev), k.to(dev), v.to(dev), torch.zeros(8, H, device=dev), bk)
    out, s = ops.rel_attention(*a, want_lse=True, **kw)
    for saved, names in ((s, ("dq", "dk", "dtable")), (s._replace(out_lo=None), ("dk", "dtable"))):
        got = dict(zip(("dq", "dk", "dv", "dtable"), ops.rel_attention_bwd(*a, out, saved, do.to(dev), **kw)))
        for n in names:
            close(got[n].double().view(want[n].shape), want[n], tol[n], n)
    assert ((got["dq"].cpu().double().view(want["dq"].shape) - want["dq"]).abs() > 2 * tol["dq"]).any(), "dq without out_lo"


def fp16_gradient_case(q, k, v, table, bk, do, H, Hk, scale, causal=False, qstart=None):
    """Gradients in fp16 against 64 bits where nothing but the operands' rounding is allowed for: every dS and P counts relative to the largest one that goes
    into the same sum, whatever the size of dO.

    dS is multiplied by a power of two that keeps the largest dS of a sum at 2^7 or above before it is rounded: one that then falls below 2^-14 is off by
    at most 2^-25, that is 2^-32 of the largest; P is multiplied by 2^14, off by at most 2^-39 there.  Nothing else is absolute (close() adds the
    result's own half step below 2^-14)."""
    from diffusion_uncertainty_amd import ops
    B, Tq, ch, Tk = q.shape[0], q.shape[1], q.shape[2] // H, k.shape[1]
    D = lambda t: None if t is None else t.to(dev)
    r = oracle.rel_attention(q, k, v, table, bk.map.cpu(), H, Hk, causal, scale, None, qstart, do)
    e = half_step(torch.float16)
    w = (2 * ((ch + 8) * r["logit"] + 8) * U + (Tk + 8) * U).max()
    ds = w + (ch + 4) * U + e * e + e
    size = lambda t: t.double().abs().max()
    ds_max = 2 * do.double().abs().reshape(B, Tq, H, ch).sum(3).max() * size(v)                       # |dP| + |D| at most
    sc = abs(scale)
    kw = dict(heads=H, kv_heads=Hk, causal=causal, scale=scale, qstart=D(qstart))
    a = (D(q), D(k), D(v), D(table), bk)
    out, s = ops.rel_attention(*a, want_lse=True, **kw)
    got = dict(zip(("dq", "dk", "dv", "dtable"), ops.rel_attention_bwd(*a, out, s, D(do), **kw)))
    n = H // Hk * Tq
    assert r["dq"].abs().max() < 65504 and r["dk"].abs().max() < 65504 and r["dv"].abs().max() < 65504
    close(got["dq"], r["dq"], r["adq"] * (ds + (Tk + 8) * U) + e * r["dq"].abs() + Tk * 2.0 ** -32 * ds_max * size(k) * sc, "dq")
    close(got["dk"], r["dk"], r["adk"] * (ds + (n + 8) * U) + e * r["dk"].abs() + n * 2.0 ** -32 * ds_max * size(q) * sc, "dk")
    close(got["dv"], r["dv"], r["adv"] * (w + e + (n + 8) * U) + e * r["dv"].abs() + n * 2.0 ** -39 * size(do), "dv")
    return got, r


@pytest.mark.parametrize("dout", [1e3, 1.0, 1e-3, 1e-5])
@pytest.mark.parametrize("Tq,Tk,H,Hk,ch", [(1, 300, 2, 1, 64), (130, 200, 2, 1, 64), (400, 400, 1, 1, 40), (200, 70, 2, 2, 128)])
def test_rel_attention_fp16_gradients_of_any_size(dout, Tq, Tk, H, Hk, ch):
    """Gradients of a mean over many tokens (far below 1) and loss-scaled ones: dq, dk, dv lose no more than their type forces."""
    from diffusion_uncertainty_amd import ops
    g = torch.Generator().manual_seed(31)
    h = torch.float16
    q, k, v, do = rnd(g, 1, Tq, H * ch, dtype=h), rnd(g, 1, Tk, Hk * ch, dtype=h), rnd(g, 1, Tk, Hk * ch, dtype=h), rnd(g, 1, Tq, H * ch, dtype=h, scale=dout)
    do[:, ::3] *= 2.0 ** -6                                                            # rows of different size share a key
    bk = ops.RelativeBuckets(8, 16, True, device=dev)
    fp16_gradient_case(q, k, v, rnd(g, 8, H, dtype=h), bk, do, H, Hk, 1.0 / math.sqrt(ch))


def test_rel_attention_fp16_gradients_past_the_types_range():
    """dS times the scale beyond 65504 with gradients that fp16 holds; a key that every query gives a probability near 2^-27; queries whose dS vary by 2^40."""
    from diffusion_uncertainty_amd import ops
    g = torch.Generator().manual_seed(32)
    h, ch = torch.float16, 64
    bk = ops.RelativeBuckets(8, 16, True, device=dev)
    zero = torch.zeros(8, 1, dtype=h)
    q, k = rnd(g, 1, 90, ch, dtype=h, scale=2.0 ** -9), rnd(g, 1, 8, ch, dtype=h, scale=2.0 ** -9)
    v, do = rnd(g, 1, 8, ch, dtype=h, scale=8.0), rnd(g, 1, 90, ch, dtype=h, scale=256.0)
    got, r = fp16_gradient_case(q, k, v, zero, bk, do, 1, 1, 64.0)
    assert r["dq"].abs().max() > 100
    q, k, v, do = (rnd(g, 1, 150, ch, dtype=h) for _ in range(4))
    q[..., 0], k[..., 0] = 8.0, 0.0
    k[:, 5::7, 0] = -14.0                                                              # scores 14 below the rest: P about 2^-27
    got, r = fp16_gradient_case(q, k, v, rnd(g, 8, 1, dtype=h), bk, do, 1, 1, 0.125)
    assert r["dv"][:, 5::7].abs().max() < 1e-3
    q, k, v, do = (rnd(g, 1, 150, ch, dtype=h) for _ in range(4))
    do[:, :75] *= 2.0 ** -20
    do[:, 75:] *= 2.0 ** 10
    do[:, 100] *= 2.0 ** 4
    fp16_gradient_case(q, k, v, rnd(g, 8, 1, dtype=h), bk, do, 1, 1, 0.125, causal=True)


# ---------------------------------------------------------------------------------------------------------- sandwich norm
def norm_case(dt, shape, post, pre, gate_rows, param_dt=torch.float32, weights=True, shifts=True, res_scale=0.7, seed=0, offset=0.0, grads=True):
    from diffusion_uncertainty_amd import ops
    g = torch.Generator().manual_seed(seed)
    D = shape[-1]
    rows = math.prod(shape[:-1])
    x, y, dr, dz = (rnd(g, *shape, dtype=dt) for _ in range(4))
    x = (x.float() * 2 + offset).to(dt)
    y = (y.float() + offset).to(dt)
    P = lambda on, s=1.0, o=0.0: (rnd(g, D, scale=s) + o).to(param_dt) if on else None
    par = dict(post_w=P(post and weights, 0.3, 1.0), post_b=P(post and shifts), pre_w=P(pre and weights, 0.3, 1.0), pre_b=P(pre and shifts),
               gate=None if gate_rows is None else rnd(g, *(() if gate_rows == 0 else (gate_rows,)), D, dtype=param_dt))
    eps = 1e-5
    L = {n: (None if t is None else t.double().requires_grad_(True)) for n, t in dict(x=x, y=y, **par).items()}
    f = lambda a: oracle.sandwich_norm(a["x"], a["y"], post, a["post_w"], a["post_b"], a["gate"], res_scale, pre, a["pre_w"], a["pre_b"], eps)
    r, z = f(L)
    D_ = lambda t: None if t is None else t.to(dev)
    kw = dict(post=post, pre=pre, res_scale=res_scale, eps=eps, **{n: D_(t) for n, t in par.items()})
    gr, gz, st = ops.sandwich_norm(D_(x), D_(y), want_stats=True, **kw)
    e = half_step(dt)
    # A row's sums are trees of depth at most 8 + 6 + 16 = 30 over terms of size t: mean and 1 / std are good to 40 u of their own size, where
    # the mean's error enters a normalised value as the offset over the deviation; 200 u covers the chain of norm, gate, sum and norm.
    absn = lambda t, kind, w, b: (t.abs() + (t.abs().mean(-1, keepdim=True) if kind == "layer" else 0)) * _rstd(t, kind, eps) * (1 if w is None else w.abs()) + (0 if b is None else b.abs())
    with torch.no_grad():
        u_mag = L["y"].abs() if post is None else absn(L["y"], post, L["post_w"], L["post_b"])
        gm = torch.ones(rows, D, dtype=torch.float64) if par["gate"] is None else L["gate"].abs().reshape(-1, D).repeat_interleave(rows // max(1, L["gate"].numel() // D), 0)
        r_mag = abs(res_scale) * L["x"].abs() + gm.reshape(shape) * u_mag
        close(gr, r, e * r.abs() + 200 * U * r_mag, "r")
        if pre is not None:
            m = r_mag + r_mag.mean(-1, keepdim=True)
            z_mag = m * _rstd(r, pre, eps) * (1 if L["pre_w"] is None else L["pre_w"].abs()) * (1 + _h(r, pre, eps).abs()) + (0 if L["pre_b"] is None else L["pre_b"].abs())
            close(gz, z, e * z.abs() + 200 * U * z_mag, "z")
        else:
            assert gz is None
    if not grads:
        return
    names = [n for n, t in L.items() if t is not None]
    outs, gs = ([r, z], [dr.double(), dz.double()]) if pre is not None else ([r], [dr.double()])
    want = dict(zip(names, torch.autograd.grad(outs, [L[n] for n in names], gs)))
    got = ops.sandwich_norm_bwd(D_(x), D_(y), st, D_(dr), D_(dz) if pre is not None else None, **kw)
    again = ops.sandwich_norm_bwd(D_(x), D_(y), st, D_(dr), D_(dz) if pre is not None else None, **kw)
    for a, b in zip(got, again):
        assert (a is None) == (b is None) and (a is None or torch.equal(a, b))
    with torch.no_grad():
        rs = _rstd(r, pre, eps) if pre else torch.ones(shape[:-1] + (1,), dtype=torch.float64)
        q = dz.double().abs() * (1 if L["pre_w"] is None else L["pre_w"].abs())
        hr = (_h(r, pre, eps).abs() + (r_mag + r_mag.mean(-1, keepdim=True)) * rs) if pre else torch.zeros(shape, dtype=torch.float64)
        t_mag = dr.double().abs() + (rs * (q + q.mean(-1, keepdim=True) + hr * (q * hr).mean(-1, keepdim=True)) if pre else 0)
        du = t_mag * gm.reshape(shape)
        eo = du * (1 if L["post_w"] is None else L["post_w"].abs())
        hy = (_h(L["y"], post, eps).abs() + (L["y"].abs().mean(-1, keepdim=True) * _rstd(L["y"], post, eps))) if post else None
        mags = dict(x=abs(res_scale) * t_mag,
                    y=du if post is None else _rstd(L["y"], post, eps) * (eo + eo.mean(-1, keepdim=True) + hy * (eo * hy).mean(-1, keepdim=True)))
        cols = lambda a: a.reshape(-1, D).sum(0)
        if post:
            mags.update(post_w=cols(du * hy), post_b=cols(du))
        if pre:
            mags.update(pre_w=cols(dz.double().abs() * hr), pre_b=cols(dz.double().abs()))
        if par["gate"] is not None:
            G = max(1, par["gate"].numel() // D)
            mags["gate"] = (t_mag * u_mag).reshape(G, rows // G, D).sum(1).reshape(par["gate"].shape)
        for n in names:
            o = getattr(got, "d" + n)
            # gradients: 300 u of the terms' magnitudes for the chain, and the depth of the column sums (chunks of rows, then chunks)
            depth = 300 + (rows // 512 + 140 if n not in ("x", "y") else 0)
            close(o, want[n], half_step(o.dtype) * want[n].abs() + depth * U * mags[n] + 1e-30, "d" + n)
        assert [n for n in ("gate", "post_w", "post_b", "pre_w", "pre_b") if getattr(got, "d" + n) is not None] == [n for n in ("gate", "post_w", "post_b", "pre_w", "pre_b") if par[n] is not None]


def _rstd(t, kind, eps):
    c = t - t.mean(-1, keepdim=True) if kind == "layer" else t
    return 1.0 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)


def _h(t, kind, eps):
    return (t - t.mean(-1, keepdim=True) if kind == "layer" else t) * _rstd(t, kind, eps)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("shape,gate_rows", [((1, 1), 0), ((3, 7), None), ((2, 5, 64), 2), ((37, 320), 0), ((4, 33, 1152), 4), ((6, 1001), 6), ((5, 4104), 0),
                                             ((3, 8192), 3)])
def test_sandwich_norm_and_gradients(dt, shape, gate_rows):
    norm_case(dt, shape, "rms", "rms", gate_rows, seed=shape[-1], shifts=False)
    norm_case(dt, shape, "layer", "layer", gate_rows, param_dt=dt, seed=shape[-1] + 1)


@pytest.mark.parametrize("post,pre,gate_rows,weights,shifts", [(None, "rms", None, True, False), ("layer", None, 0, True, True), (None, None, 3, False, False),
                                                               ("rms", "layer", 0, False, False), ("layer", "rms", 12, True, True)])
def test_sandwich_norm_forms(post, pre, gate_rows, weights, shifts):
    for dt in (torch.float32, torch.bfloat16):
        norm_case(dt, (12, 200), post, pre, gate_rows, weights=weights, shifts=shifts)


@pytest.mark.parametrize("shape,gate_rows", [((1500, 96), 0), ((1500, 96), 3), ((1500, 96), 500), ((1500, 96), 1500), ((1, 1025, 40), 1)])
def test_sandwich_norm_gradient_chunks(shape, gate_rows):
    """More rows than chunks of the backward pass: chunks inside a sample, chunks of whole samples, samples of one row."""
    norm_case(torch.float32, shape, "rms", "layer", gate_rows)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("D,gate_rows", [(3, 211), (64, 0), (65, 422), (127, 1), (128, 2), (130, 0), (250, 422), (257, 0), (511, 2), (513, 211), (2049, 0), (4096, 2)])
def test_sandwich_norm_units_of_every_width(dt, D, gate_rows):
    """Rows held by 16 or 32 lanes, a wavefront, up to 16 wavefronts, and the widths around each border; 422 rows."""
    norm_case(dt, (422, D), "layer", "rms", gate_rows, seed=D)


def test_sandwich_norm_large_offset_and_constant_rows():
    """LayerNorm of rows whose mean is far from zero (two-pass variance) and of constant rows (variance 0: 1 / std = eps^-1/2)."""
    from diffusion_uncertainty_amd import ops
    norm_case(torch.float32, (9, 512), "layer", "layer", 0, offset=100.0, grads=False)
    x = torch.full((2, 512), 3.0, device=dev)
    r, z = ops.sandwich_norm(x, x, post="layer", pre="layer", eps=1e-6)
    assert torch.equal(r, x) and (z == 0).all()


def test_sandwich_norm_in_place_and_empty():
    from diffusion_uncertainty_amd import _lib, ops
    z0 = torch.zeros(0, 64, device=dev)
    w = torch.ones(64, device=dev)
    r, z, st = ops.sandwich_norm(z0, z0, post_w=w, gate=w, want_stats=True)
    assert r.shape == (0, 64) and z.shape == (0, 64)
    g = ops.sandwich_norm_bwd(z0, z0, st, z0, z0, post_w=w, gate=w)
    assert (g.dpost_w == 0).all() and (g.dgate == 0).all() and g.dpre_w is None
    # the C entry allows r over x and z over y
    import ctypes
    gen = torch.Generator().manual_seed(0)
    x, y = rnd(gen, 5, 100).to(dev), rnd(gen, 5, 100).to(dev)
    r, z = ops.sandwich_norm(x, y)
    a = _lib.SandwichNormArgs(x=x.data_ptr(), y=y.data_ptr(), dtype=0, param_dtype=0, rows=5, D=100, post=1, pre=1, res_scale=1.0, eps=1e-6,
                              r=x.data_ptr(), z=y.data_ptr())
    _lib.check(_lib.lib().dua_sandwich_norm(ctypes.byref(a), ops._stream()), "dua_sandwich_norm")
    assert torch.equal(x, r) and torch.equal(y, z)


def test_sandwich_norm_empty_batch_with_a_gate_for_each_sample():
    """No samples, no gate rows: nothing to do, zeros for the parameters' gradients."""
    from diffusion_uncertainty_amd import ops
    x, gate, w = torch.zeros(0, 7, 64, device=dev), torch.zeros(0, 64, device=dev), torch.ones(64, device=dev)
    r, z, st = ops.sandwich_norm(x, x, post_w=w, pre_w=w, gate=gate, want_stats=True)
    assert r.shape == z.shape == (0, 7, 64) and st.shape == (0, 4)
    g = ops.sandwich_norm_bwd(x, x, st, x, x, post_w=w, pre_w=w, gate=gate)
    assert g.dx.shape == (0, 7, 64) and g.dgate.shape == (0, 64) and (g.dpost_w == 0).all() and (g.dpre_w == 0).all()
    with pytest.raises(ValueError):
        ops.sandwich_norm(torch.zeros(2, 64, device=dev), torch.zeros(2, 64, device=dev), gate=gate)


# --------------------------------------------------------------------------------------------------------- token logprobs
def logprob_case(x, ids, k, t=1.0, grads=True, seed=0):
    """x [rows, V] on the CPU in its type.  A row's sums: chains of V / 256 / parts groups of up to 8 and trees of depth 14; each exponential is good
    to 4 u + |x - m| t 2 u relative."""
    from diffusion_uncertainty_amd import ops
    rows, V = x.shape
    xd = x.double().requires_grad_(True)
    lp, ent, lse, top, tlp, l = oracle.token_logprobs(xd, ids, k, t)
    o = ops.token_logprobs(x.to(dev), None if ids is None else ids.to(dev), k=k, inv_temperature=t)
    live, l = lse.detach() > -math.inf, l.detach()
    with torch.no_grad():
        p = torch.exp(l)
        span = torch.where(p > 1e-40, l.abs(), torch.zeros_like(l)).max(1).values                 # logits that count
        g = ((V / 256 + 30) + 4 * span) * U                                                # relative error of s, absolute of log s
        lse, lp, tlp = (torch.where(torch.isnan(a), a, a.float().double()) for a in (lse, lp, tlp))   # (past fp32's range: infinite)
        close(o.lse, lse, g + 4 * U * lse.abs().nan_to_num(posinf=0.0) + 1e-30, "lse")
        close(o.entropy, ent, g * (2 + 2 * ent.abs() + span.clamp(max=4)) + 1e-30, "entropy")
        close(o.logprob, lp, g + 4 * U * lp.abs().nan_to_num(posinf=0.0) + 1e-30, "logprob")
        if k:
            assert torch.equal(o.top_ids.cpu(), top), "alternatives"
            close(o.top_logprobs, tlp, (g[:, None] + 4 * U * tlp.abs().nan_to_num(posinf=0.0)) + 1e-30, "top_logprobs")
    if not grads:
        return o
    gen = torch.Generator().manual_seed(seed + 1)
    gl, gh, gt = rnd(gen, rows), rnd(gen, rows), rnd(gen, rows, k)
    with torch.no_grad():
        hot = torch.zeros(rows, V, dtype=torch.float64)
        ok = (ids >= 0) & (ids < V)
        gle = torch.where(ok, gl.double(), 0.0)
        hot.scatter_add_(1, torch.where(ok, ids, 0)[:, None], gle[:, None])
        hot.scatter_add_(1, top, gt.double())
        A = gle + gt.double().sum(1)
        Aabs = gle.abs() + gt.double().abs().sum(1)
        pl = torch.where(p > 0, p * torch.where(p > 0, l, 0.0), 0.0)
        want = t * (hot - p * A[:, None] - gh.double()[:, None] * (pl + p * ent[:, None]))
        want = torch.where(live[:, None], want, 0.0)
        mag = t * (hot.abs() + p * Aabs[:, None] + gh.double().abs()[:, None] * (pl.abs() + p * ent[:, None]))
        mag = torch.where(live[:, None], mag, 0.0)
    got = ops.token_logprobs_bwd(x.to(dev), ids.to(dev), o, dlogprob=gl.to(dev), dentropy=gh.to(dev), dtop=gt.to(dev) if k else None, inv_temperature=t)
    tol = half_step(x.dtype) * want.abs() + (3 * g[:, None] + (k + 40) * U + 2 * U * l.abs().nan_to_num(posinf=0.0)) * mag
    close(got, want, tol + 1e-37, "dlogits")
    xi = x.to(dev)
    assert torch.equal(ops.token_logprobs_bwd(xi, ids.to(dev), o, gl.to(dev), gh.to(dev), gt.to(dev) if k else None, t, out=xi), got) and torch.equal(xi, got)
    return o


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows,V,k", [(1, 1, 1), (3, 2, 2), (5, 63, 8), (7, 1000, 20), (300, 257, 5), (2, 4099, 64), (3, 40001, 20), (2, 65536, 0)])
def test_token_logprobs_and_gradient(dt, rows, V, k):
    g = torch.Generator().manual_seed(V)
    x = rnd(g, rows, V, scale=2.5, dtype=dt)
    logprob_case(x, torch.randint(0, V, (rows,), generator=g), k, seed=V)


@pytest.mark.parametrize("dt", DTYPES)
def test_token_logprobs_temperature_and_masks(dt):
    g = torch.Generator().manual_seed(5)
    x = rnd(g, 12, 5000, scale=3.0, dtype=dt)
    low = torch.finfo(dt).min
    x[0, 1:] = -math.inf                       # one token left
    x[1, ::2] = -math.inf
    x[2, 100:] = low                           # masks of the type's lowest value
    x[3, :] = low                              # ... everywhere: uniform
    x[4, :] = 0.0                              # equal logits: alternatives 0, 1, 2, ...
    x[5, 4990:] = -math.inf
    x[6, :3000] = x[6, 0]
    x[7] = torch.sort(x[7].float()).values.to(dt)                         # every element beats all before it
    x[8, ::3], x[8, 1::3] = 0.0, -0.0          # equal: ties by index, not by sign
    x[8, 2::3] = -1.0
    x[9, 7:] = -math.inf                       # fewer finite values than alternatives
    ids = torch.tensor([0, 1, 50, 7, 4999, 3, 1, 4999, 4, 2, -100, 5000])
    logprob_case(x, ids, 20, t=0.8)
    logprob_case(x, ids, 0, t=1.7)


@pytest.mark.parametrize("dt", DTYPES)
def test_token_logprobs_of_decided_rows_keep_their_sign(dt):
    """Rows that one token decides: no log probability above 0, no entropy below it (a square root or log(1 - p) of them would be NaN)."""
    from diffusion_uncertainty_amd import ops
    g = torch.Generator().manual_seed(14)
    for V in (7, 1001, 40000):
        x = rnd(g, 64, V, dtype=dt)
        best = torch.randint(0, V, (64,), generator=g)
        lead = torch.linspace(0, 40, 64)
        x[torch.arange(64), best] = (x.float().max(1).values + lead + 5.0 * torch.rand(64, generator=g)).to(dt)
        x[32:] = (x[32:].float() + 300.0 * torch.rand(32, 1, generator=g)).to(dt)
        for t in (1.0, 0.7, 3.1):
            o = logprob_case(x, best, min(V, 5), t=t, grads=False)
            assert (o.logprob <= 0).all() and (o.top_logprobs <= 0).all() and (o.entropy >= 0).all(), (V, t, float(o.logprob.max()), float(o.entropy.min()))


def test_token_logprobs_huge_offsets():
    g = torch.Generator().manual_seed(6)
    x = rnd(g, 4, 700) + torch.tensor([3e4, -3e4, 1e30, -2e38])[:, None]
    logprob_case(x, torch.tensor([1, 2, 3, 4]), 5)


def test_token_logprobs_rows_without_a_distribution():
    from diffusion_uncertainty_amd import ops
    x = torch.randn(5, 3000, generator=torch.Generator().manual_seed(1))
    x[0] = -math.inf
    x[1, 5] = math.nan
    x[2, 7] = math.inf
    x[3, [3, 9]] = math.nan
    ids = torch.zeros(5, dtype=torch.int64)
    o = ops.token_logprobs(x.to(dev), ids.to(dev), k=4)
    c = lambda t: t.cpu()
    assert c(o.logprob)[0] == -math.inf and c(o.lse)[0] == -math.inf and c(o.entropy)[0] == 0 and c(o.top_ids)[0].tolist() == [0, 1, 2, 3]
    assert (c(o.top_logprobs)[0] == -math.inf).all()
    for i in (1, 2, 3):
        assert c(o.logprob)[i].isnan() and c(o.entropy)[i].isnan() and c(o.lse)[i].isnan()
    assert c(o.top_ids)[1, 0] == 5 and c(o.top_ids)[2, 0] == 7 and c(o.top_ids)[3, :2].tolist() == [3, 9]
    assert torch.isfinite(c(o.logprob)[4]) and torch.isfinite(c(o.entropy)[4])
    d = ops.token_logprobs_bwd(x.to(dev), ids.to(dev), o, dlogprob=torch.ones(5, device=dev), dentropy=torch.ones(5, device=dev)).cpu()
    assert (d[0] == 0).all() and d[1].isnan().all() and torch.isfinite(d[4]).all()


@pytest.mark.parametrize("dt", DTYPES)
def test_token_logprobs_long_rows_in_parts(dt):
    """Few long rows are cut into parts: parts without finite values, of the type's lowest value, with equal values, beside ordinary ones; NaN."""
    g = torch.Generator().manual_seed(12)
    V = 40000
    x = rnd(g, 7, V, scale=2.0, dtype=dt)
    low = torch.finfo(dt).min
    x[0, 5000:] = -math.inf
    x[1, 100:] = low                                   # a filter that kept a hundred tokens
    x[2, :] = low
    x[3, :] = 1.5
    x[4, 30000:] = x[4, :10000]
    x[5, :39990] = -math.inf
    ids = torch.tensor([3, 39999, 20000, 39998, 30001, 39995, 12345])
    logprob_case(x, ids, 20)
    from diffusion_uncertainty_amd import ops
    y = rnd(g, 4, V, scale=2.0, dtype=dt)
    y[0, 33333] = math.nan
    y[1, 22222] = math.inf
    y[2] = -math.inf
    o = ops.token_logprobs(y.to(dev), k=3)
    assert o.lse[:2].isnan().all() and o.entropy[:2].isnan().all() and o.lse[2] == -math.inf and o.entropy[2] == 0 and torch.isfinite(o.lse[3])
    assert o.top_ids[0, 0] == 33333 and o.top_ids[1, 0] == 22222 and o.top_ids[2].tolist() == [0, 1, 2]
    if dt == torch.float32:                            # offsets past the floating reference, alone and beside ordinary parts
        z = rnd(g, 3, V)
        z[0] += 1e30
        z[1, 35000:] -= 3e9
        z[2, 10] = 2e9
        logprob_case(z, torch.tensor([5, 6, 10]), 5)


@pytest.mark.parametrize("dt", DTYPES)
def test_token_logprobs_many_long_rows_in_parts(dt):
    """More than 255 rows of 192 KB and beyond, cut into parts: equal rows give equal bits."""
    from diffusion_uncertainty_amd import ops
    g = torch.Generator().manual_seed(13)
    V = 100003 if dt != torch.float32 else 50003
    base = rnd(g, 8, V, scale=2.0, dtype=dt)
    base[1, 40000:] = -math.inf
    ids = torch.randint(0, 40000, (8,), generator=g)
    logprob_case(base, ids, 8, grads=False)
    few = ops.token_logprobs(base.to(dev), ids.to(dev), k=8)
    r = torch.arange(260) % 8
    many = ops.token_logprobs(base.to(dev)[r.to(dev)], ids[r].to(dev), k=8)
    lp, ent, lse, top, tlp, l = oracle.token_logprobs(base.double(), ids, 8, 1.0)
    assert torch.equal(many.top_ids.cpu(), top[r])
    for a, b in ((many.logprob, lp), (many.entropy, ent), (many.lse, lse)):
        assert torch.equal(a.cpu()[:8].repeat(33)[:260], a.cpu()), "equal rows, equal bits"
        # two orders of a sum of V / 1024 terms a thread and trees: V / 256 + 30 half steps, 4 for each unit of the largest logit that counts (40)
        close(a, b[r], (V / 256 + 30 + 160) * U * (2 + 2 * b[r].abs()), "many")
    assert (many.logprob - few.logprob[r.to(dev)]).abs().max() < 1e-4


def test_token_logprobs_views_and_partial_gradients():
    """A slice of a padded vocabulary (row stride > V, rows not 16-byte aligned), leading dimensions, missing gradients, no ids, repeated ids."""
    from diffusion_uncertainty_amd import ops
    g = torch.Generator().manual_seed(9)
    for dt in DTYPES:
        full = rnd(g, 2, 6, 1031, dtype=dt).to(dev)
        x, ids = full[..., 1:1025], torch.randint(0, 1024, (2, 6), generator=g).to(dev)
        a, b = ops.token_logprobs(x, ids, k=3), ops.token_logprobs(x.contiguous(), ids, k=3)
        for p, q in zip(a, b):
            assert torch.equal(p, q) or (p - q).abs().max() < 1e-5                         # (the groups fall differently: sums may)
        gl = rnd(g, 2, 6).to(dev)
        d = ops.token_logprobs_bwd(x, ids, a, dlogprob=gl)
        want = gl[..., None] * (torch.nn.functional.one_hot(ids, 1024) - torch.softmax(x.float(), -1))
        assert (d.float() - want).abs().max() < 4 * half_step(dt) + 1e-5
        assert (ops.token_logprobs_bwd(x, None, a) == 0).all()
        into = torch.full((2, 6, 1031), 7.0, device=dev, dtype=dt)
        ops.token_logprobs_bwd(x, ids, a, dlogprob=gl, out=into[..., 2:1026])
        assert torch.equal(into[..., 2:1026], d) and (into[..., :2] == 7).all() and (into[..., 1026:] == 7).all()
        # the given token is also the best alternative: it gets both gradients
        best = a.top_ids[..., 0].contiguous()
        gt = rnd(g, 2, 6, 3).to(dev)
        s = ops.token_logprobs(x, best, k=3)
        both = ops.token_logprobs_bwd(x, best, s, dlogprob=gl, dtop=gt)
        merged = gt.clone()
        merged[..., 0] += gl
        alone = ops.token_logprobs_bwd(x, best, s, dtop=merged)
        assert (both.float() - alone.float()).abs().max() < 4 * half_step(dt) * 4 + 1e-5
    assert (ops.token_logprobs(x).logprob == 0).all() and ops.token_logprobs(x).top_ids is None
    e = ops.token_logprobs(x[:0], ids[:0], k=2)
    assert e.logprob.shape == (0, 6) and e.top_ids.shape == (0, 6, 2)
    assert ops.token_logprobs_bwd(x[:0], ids[:0], e).shape == (0, 6, 1024)


def test_token_logprobs_gradient_against_differences():
    from diffusion_uncertainty_amd import ops
    g = torch.Generator().manual_seed(11)
    x, ids = rnd(g, 6, 301, scale=2.0), torch.randint(0, 301, (6,), generator=g)
    gl, gh, gt = rnd(g, 6), rnd(g, 6), rnd(g, 6, 4)
    o = ops.token_logprobs(x.to(dev), ids.to(dev), k=4, inv_temperature=1.3)
    grad = ops.token_logprobs_bwd(x.to(dev), ids.to(dev), o, gl.to(dev), gh.to(dev), gt.to(dev), 1.3).cpu().double()
    top = o.top_ids.cpu()

    def f(z):
        lp, ent, _, _, _, l = oracle.token_logprobs(z, ids, 4, 1.3)
        return ((lp * gl).sum() + (ent * gh).sum() + (l.gather(1, top) * gt).sum()).item()

    for _ in range(3):
        d = torch.randn(x.shape, generator=g, dtype=torch.float64)
        diff = (f(x.double() + 1e-5 * d) - f(x.double() - 1e-5 * d)) / 2e-5
        assert abs(diff - (grad * d).sum().item()) < 1e-5 * (grad * d).abs().sum().item() + 1e-6


# ------------------------------------------------------------------------------------------- refusals, streams, graphs, together
def test_token_operator_refusals():
    from diffusion_uncertainty_amd import ops
    z = lambda *s, dt=torch.float32: torch.zeros(*s, device=dev, dtype=dt)
    bk = ops.RelativeBuckets(8, 16, True, device=dev)
    q, table = z(1, 4, 64), z(8, 2)
    bad = [(TypeError, lambda: ops.rel_attention(z(1, 4, 64, dt=torch.float64), q, q, table, bk, heads=2)),
           (TypeError, lambda: ops.rel_attention(q, z(1, 4, 64, dt=torch.float16), q, table, bk, heads=2)),
           (TypeError, lambda: ops.rel_attention(q, q, q, z(8, 2, dt=torch.float16), bk, heads=2)),
           (ValueError, lambda: ops.rel_attention(q, q, q, z(7, 2), bk, heads=2)),
           (ValueError, lambda: ops.rel_attention(q, q, q, table, bk, heads=3)),
           (ValueError, lambda: ops.rel_attention(q, q, z(1, 5, 64), table, bk, heads=2)),
           (ValueError, lambda: ops.rel_attention(z(1, 64, 4).transpose(1, 2), q, q, table, bk, heads=2)),
           (ValueError, lambda: ops.rel_attention(q, q, q, table, torch.zeros(33), heads=2)),
           (TypeError, lambda: ops.rel_attention(q, q, q, table, bk, heads=2, klen=torch.zeros(1, device=dev, dtype=torch.int64))),
           (ValueError, lambda: ops.rel_attention(q, q, q, table, bk, heads=2, klen=torch.zeros(2, device=dev, dtype=torch.int32))),
           (RuntimeError, lambda: ops.rel_attention(z(1, 4, 272), z(1, 4, 272), z(1, 4, 272), table, bk, heads=2)),
           (RuntimeError, lambda: ops.rel_attention(z(1, 4, 66), z(1, 4, 66), z(1, 4, 66), table, bk, heads=2)),
           (RuntimeError, lambda: ops.rel_attention(torch.zeros(1, 4, 64), q, q, table, bk, heads=2)),
           (TypeError, lambda: ops.rel_attention_bwd(q, q, q, table, bk, q, z(1, 2, 4), q, heads=2)),
           (ValueError, lambda: ops.rel_attention_bwd(q, q, q, table, bk, q, ops.RelAttentionSaved(z(1, 2, 5), None), q, heads=2)),
           (ValueError, lambda: ops.sandwich_norm(z(4, 8), z(4, 9))),
           (ValueError, lambda: ops.sandwich_norm(z(4, 8), z(4, 8), post=None, post_w=z(8))),
           (ValueError, lambda: ops.sandwich_norm(z(4, 8), z(4, 8), post="batch")),
           (ValueError, lambda: ops.sandwich_norm(z(4, 8), z(4, 8), gate=z(3, 8))),
           (ValueError, lambda: ops.sandwich_norm(z(8, 4).t(), z(4, 8))),
           (TypeError, lambda: ops.sandwich_norm(z(4, 8), z(4, 8), post_w=z(8), pre_w=z(8, dt=torch.float16))),
           (RuntimeError, lambda: ops.sandwich_norm(z(2, 8193), z(2, 8193))),
           (ValueError, lambda: ops.sandwich_norm_bwd(z(4, 8), z(4, 8), z(4, 4), z(4, 8), z(4, 8), pre=None)),
           (ValueError, lambda: ops.token_logprobs(z(4, 8), k=9)),
           (ValueError, lambda: ops.token_logprobs(z(4, 100), k=65)),
           (ValueError, lambda: ops.token_logprobs(z(4, 8), inv_temperature=0.0)),
           (ValueError, lambda: ops.token_logprobs(z(4, 8), inv_temperature=math.nan)),
           (TypeError, lambda: ops.token_logprobs(z(4, 8), torch.zeros(4, device=dev, dtype=torch.int32))),
           (ValueError, lambda: ops.token_logprobs(z(4, 8), torch.zeros(3, device=dev, dtype=torch.int64))),
           (ValueError, lambda: ops.token_logprobs(z(1, 8).expand(4, 8))),
           (ValueError, lambda: ops.token_logprobs(z(8, 4).t()))]
    for exc, call in bad:
        with pytest.raises(exc):
            call()
    o = ops.token_logprobs(z(4, 8), torch.zeros(4, device=dev, dtype=torch.int64))
    with pytest.raises(ValueError):
        ops.token_logprobs_bwd(z(4, 8), None, o, dlogprob=z(4))
    with pytest.raises(ValueError):
        ops.token_logprobs_bwd(z(4, 8), None, o, dtop=z(4, 1))


class Block:
    """Two blocks of a small token denoiser from the public operators: attention with the bucketed bias, sandwich norms, the library's own
    projections, the answer's log probabilities; the mean negative log probability plus its entropy as the loss, gradients by hand."""

    def __init__(self, seed, B=2, T=50, H=2, ch=32, V=1112):
        from diffusion_uncertainty_amd import ops
        g = torch.Generator().manual_seed(seed)
        D = H * ch
        self.ops, self.shape, self.H = ops, (B, T, D), H
        w = lambda *s: (torch.randn(*s, generator=g) / math.sqrt(s[-1])).to(dev)
        self.x, self.ids = torch.randn(B, T, D, generator=g).to(dev), torch.randint(0, V, (B, T), generator=g).to(dev)
        self.wqkv, self.wo, self.head = w(3 * D, D), w(D, D), w(V, D)
        self.table, self.pw, self.qw = torch.randn(8, H, generator=g).to(dev), w(D) + 1, w(D) + 1
        self.gate = torch.randn(B, D, generator=g).to(dev)
        self.klen = torch.tensor([T, T // 2], dtype=torch.int32, device=dev)
        self.buckets = ops.RelativeBuckets(8, 16, True, device=dev)
        self.kw = dict(post="rms", post_w=self.pw, gate=self.gate, res_scale=0.8, pre="rms", pre_w=self.qw)

    def step(self):
        ops, (B, T, D) = self.ops, self.shape
        lin = lambda a, w: ops.gemm(a.reshape(B * T, -1), w).view(B, T, -1)
        qkv = lin(self.x, self.wqkv)
        q, k, v = qkv[..., :D], qkv[..., D:2 * D], qkv[..., 2 * D:]
        att, lse = ops.rel_attention(q, k, v, self.table, self.buckets, heads=self.H, klen=self.klen, want_lse=True)
        y = lin(att, self.wo)
        r, z, st = ops.sandwich_norm(self.x, y, want_stats=True, **self.kw)
        logits = lin(z, self.head)
        o = ops.token_logprobs(logits, self.ids, k=3)
        mask, _ = ops.quantile_mask(o.entropy.view(B, T), 0.9)
        n = B * T
        dl = ops.token_logprobs_bwd(logits, self.ids, o, dlogprob=torch.full((B, T), -1.0 / n, device=dev), dentropy=torch.full((B, T), 0.1 / n, device=dev))
        T_ = lambda w: w.t().contiguous()
        dz = lin(dl, T_(self.head))
        g = ops.sandwich_norm_bwd(self.x, y, st, torch.zeros_like(r), dz, **self.kw)
        datt = lin(g.dy, T_(self.wo))
        dq, dk, dv, dtable = ops.rel_attention_bwd(q, k, v, self.table, self.buckets, att, lse, datt, heads=self.H, klen=self.klen)
        dx = g.dx + lin(torch.cat([dq, dk, dv], 2), T_(self.wqkv))
        return dict(r=r, z=z, logprob=o.logprob, entropy=o.entropy, top=o.top_ids, mask=mask, dx=dx, dtable=dtable, dpw=g.dpost_w, dqw=g.dpre_w, dgate=g.dgate)


def test_operators_together_against_autograd_in_64_bits():
    b = Block(1)
    got = b.step()
    B, T, D = b.shape
    H, ch = b.H, D // b.H
    L = {n: getattr(b, n).cpu().double().requires_grad_(True) for n in ("x", "table", "pw", "qw", "gate")}
    W = {n: getattr(b, n).cpu().double() for n in ("wqkv", "wo", "head")}
    q, k, v = (t.view(B, T, H, ch).transpose(1, 2) for t in (L["x"] @ W["wqkv"].T).split(D, 2))
    rel = (torch.arange(T)[None] - torch.arange(T)[:, None]).clamp(-16, 16) + 16
    s = q @ k.transpose(2, 3) / math.sqrt(ch) + L["table"][b.buckets.map.cpu().long()[rel]].permute(2, 0, 1)
    s = s.masked_fill(torch.arange(T) >= b.klen.cpu()[:, None, None, None], -math.inf)
    y = (torch.softmax(s, -1) @ v).transpose(1, 2).reshape(B, T, D) @ W["wo"].T
    r, z = oracle.sandwich_norm(L["x"], y, "rms", L["pw"], None, L["gate"], 0.8, "rms", L["qw"], None, 1e-6)
    lp, ent, lse, _, _, _ = oracle.token_logprobs((z @ W["head"].T).view(B * T, -1), b.ids.cpu().view(-1), 3, 1.0)
    loss = (-lp + 0.1 * ent).mean()
    gx, gt, gpw, gqw, gg = torch.autograd.grad(loss, [L[n] for n in ("x", "table", "pw", "qw", "gate")])
    for n, want in (("r", r), ("z", z), ("logprob", lp.view(B, T)), ("entropy", ent.view(B, T)), ("dx", gx), ("dtable", gt), ("dpw", gpw), ("dqw", gqw), ("dgate", gg)):
        err = (got[n].cpu().double() - want.detach()).abs().max() / want.detach().abs().max()
        # fp32 throughout: chains of up to 64 + 64 + 1112 products between input and loss and back, 2^-24 each at most
        assert err < 1300 * U, (n, float(err))
    u = got["entropy"].cpu()
    assert torch.equal(got["mask"].cpu().bool(), u > torch.quantile(u, 0.9, dim=1, keepdim=True))


def test_offsets_past_32_bits():
    """Slots of a cache and rows of logits 2^23 elements apart, a stream of more than 2^31 elements: the same bits as from small tensors."""
    from diffusion_uncertainty_amd import ops
    g = torch.Generator().manual_seed(12)
    T, far = 300, 1 << 23
    base = torch.empty(T * far, device=dev, dtype=torch.bfloat16)
    at = lambda c, w: base.as_strided((1, T, w), (T * far, far, 1), c)
    k, v, q, do = (rnd(g, 1, T, 128, dtype=torch.bfloat16).to(dev) for _ in range(4))
    kf, vf = at(0, 128).copy_(k), at(128, 128).copy_(v)
    bk, table = ops.RelativeBuckets(8, 16, True, device=dev), rnd(g, 8, 2).to(dev)
    for n in (1, T):
        assert torch.equal(ops.rel_attention(q[:, :n], kf, vf, table, bk, heads=2), ops.rel_attention(q[:, :n], k, v, table, bk, heads=2))
    out, s = ops.rel_attention(q, k, v, table, bk, heads=2, want_lse=True)
    for a, b in zip(ops.rel_attention_bwd(q, kf, vf, table, bk, out, s, do, heads=2), ops.rel_attention_bwd(q, k, v, table, bk, out, s, do, heads=2)):
        assert torch.equal(a, b)
    x, ids, gl = rnd(g, T, 1000, dtype=torch.bfloat16).to(dev), torch.randint(0, 1000, (T,), generator=g).to(dev), rnd(g, T).to(dev)
    xf, into = at(256, 1000)[0].copy_(x), at(1264, 1000)[0]
    a, b = ops.token_logprobs(xf, ids, k=4), ops.token_logprobs(x, ids, k=4)
    for m, n in zip(a, b):
        assert torch.equal(m, n)
    assert torch.equal(ops.token_logprobs_bwd(xf, ids, a, dlogprob=gl, out=into), ops.token_logprobs_bwd(x, ids, b, dlogprob=gl))
    del base, kf, vf, xf, into
    rows, D = (1 << 18) + 5, 8192
    x, y = (torch.empty(rows, D, device=dev, dtype=torch.bfloat16).normal_() for _ in range(2))
    r, z, st = ops.sandwich_norm(x, y, want_stats=True)
    r8, z8, st8 = ops.sandwich_norm(x[-8:], y[-8:], want_stats=True)
    assert torch.equal(r[-8:], r8) and torch.equal(z[-8:], z8) and torch.equal(st[-8:], st8)
    del r, z
    d, d8 = ops.sandwich_norm_bwd(x, y, st, y, x), ops.sandwich_norm_bwd(x[-8:], y[-8:], st8, y[-8:], x[-8:])
    assert torch.equal(d.dx[-8:], d8.dx) and torch.equal(d.dy[-8:], d8.dy)


def test_wide_heads_and_rows_in_a_graph():
    """Kernels with more than 64 KB of LDS (heads of 128, backward norms of 8192 columns) captured and replayed."""
    from diffusion_uncertainty_amd import ops
    g = torch.Generator().manual_seed(6)
    q, k, v, do = (rnd(g, 1, 150, 256, dtype=torch.bfloat16).to(dev) for _ in range(4))
    x, y, dr, dz = (rnd(g, 40, 8192).to(dev) for _ in range(4))
    w = rnd(g, 8192).to(dev)
    bk, table = ops.RelativeBuckets(8, 16, True, device=dev), rnd(g, 8, 2).to(dev)

    def step():
        out, s = ops.rel_attention(q, k, v, table, bk, heads=2, want_lse=True)
        r, z, st = ops.sandwich_norm(x, y, post_w=w, pre_w=w, gate=w, want_stats=True)
        return [out, *ops.rel_attention_bwd(q, k, v, table, bk, out, s, do, heads=2), r, z] + [
            t for t in ops.sandwich_norm_bwd(x, y, st, dr, dz, post_w=w, pre_w=w, gate=w) if t is not None]

    step()
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        o = step()
    for i in range(3):
        q.mul_(0.9)
        x.add_(0.1)
        gr.replay()
        want = step()
        torch.cuda.synchronize()
        for a, b in zip(o, want):
            assert torch.equal(a, b), i


def test_operators_on_another_stream_two_at_a_time_and_in_a_graph():
    b, c = Block(2), Block(3)
    want, want_c = b.step(), c.step()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (s1, s2):
        s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s1):
        g1 = b.step()
    with torch.cuda.stream(s2):
        g2 = c.step()
    torch.cuda.synchronize()
    for n in want:
        assert torch.equal(g1[n], want[n]) and torch.equal(g2[n], want_c[n]), n
    graphs = []
    for m in (b, c):
        s1.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s1):
            m.step()
        torch.cuda.current_stream().wait_stream(s1)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            o = m.step()
        graphs.append((gr, o, m))
    for i in range(3):
        for gr, o, m in graphs:
            m.x.mul_(1.0 + 0.1 * i)
            gr.replay()
        torch.cuda.synchronize()
        for gr, o, m in graphs:
            eager = m.step()
            torch.cuda.synchronize()
            for n in eager:
                assert torch.equal(o[n], eager[n]), (i, n)
