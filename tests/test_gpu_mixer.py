"""Token-mixer operators on the device against their definitions in 64 bits: head norm + rotation, the 4-bit KV cache, linear
attention with a decay per head.  Tolerances are sums of rounding errors: half a step of the type of every rounding on the way,
times the magnitudes that tests/mixer_ref.py returns beside the result."""
import numpy as np
import pytest

import mixer_ref as ref
from gpu_util import rel_l2, torch_cuda
from mixer_ref import U16, U32

pytestmark = pytest.mark.gpu

DTYPES = ["f32", "bf16"]


def to_dev(a, dtype="f32"):
    torch = torch_cuda()
    t = torch.from_numpy(np.ascontiguousarray(a, np.float32)).cuda()
    return t.bfloat16() if dtype == "bf16" else t


def host(t):
    return t.float().cpu().numpy()


def ints(a):
    torch = torch_cuda()
    return torch.tensor(list(a), dtype=torch.int32, device="cuda")


def rows(rng, shape, dtype):
    a = rng.standard_normal(shape).astype(np.float32)
    return ref.bf16(a) if dtype == "bf16" else a


def within(got, want, tol, what=""):
    bad = ~(np.abs(got.astype(np.float64) - want) <= tol)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} values off, worst {np.nanmax(np.abs(got - want) / np.maximum(tol, 1e-300)):.3g} tolerances"


# ------------------------------------------------------------------------------------------------ head norm + rotation

def check_norm_rope(T, nh, nkv, hd, rot, rot_at, halves, dtype, norm=True, weights=True, seed=0, strided=False):
    from microkimi_amd import mixer
    torch = torch_cuda()
    rng = np.random.default_rng(seed)
    qn, kn = rows(rng, (T, nh, hd), dtype) * 3, rows(rng, (T, nkv, hd), dtype)
    qn, kn = (ref.bf16(qn), ref.bf16(kn)) if dtype == "bf16" else (qn, kn)
    wq, wk = (rng.standard_normal(hd).astype(np.float32) for _ in range(2)) if weights else (None, None)
    n_pos = 5000
    cos, sin = mixer.rope_table(n_pos, rot) if rot else (None, None)
    pos = rng.integers(0, n_pos, T)
    q, k = to_dev(qn, dtype), to_dev(kn, dtype)
    if strided:  # slices of one fused row with something in between
        fused = torch.full((T, nh + nkv + 3, hd), float("nan"), dtype=q.dtype, device="cuda")
        fused[:, :nh], fused[:, nh + 1:nh + 1 + nkv] = q, k
        q, k = fused[:, :nh], fused[:, nh + 1:nh + 1 + nkv]
    qo, ko = mixer.qk_norm_rope(q, k, cos, sin, ints(pos) if rot else None, None if wq is None else to_dev(wq), None if wk is None else to_dev(wk), eps=1e-5,
                                norm=norm, rot_at=rot_at, halves=halves)
    at = hd - rot if rot_at is None else rot_at
    for got, x, w in ((qo, qn, wq), (ko, kn, wk)):
        want, mag = ref.norm_rope(x, w, 1e-5, norm, host(cos) if rot else None, host(sin) if rot else None, pos, at, halves)
        # sum of hd squares (at most 8 + 6 additions a value deep, 2 half steps a square), mean, eps, root, quotient: each enters
        # once; two products; the rotation's two products and one sum: under 32 half steps of the pair's magnitude
        tol = 32 * U32 * mag + (U16 * (np.abs(want) + 32 * U32 * mag) if dtype == "bf16" else 0)
        within(host(got), want, tol + 1e-37, f"T {T} hd {hd}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("T,nh,nkv,hd,rot,rot_at", [(1, 96, 96, 192, 64, None), (5, 64, 8, 128, 128, None), (3, 7, 1, 64, 32, 0), (2, 1, 1, 8, 0, None),
                                                    (4, 3, 2, 256, 96, 64), (2, 5, 2, 512, 64, 448), (1, 2, 2, 16, 16, 0), (9, 33, 3, 40, 16, 8)])
def test_norm_rope(T, nh, nkv, hd, rot, rot_at, halves, dtype):
    check_norm_rope(T, nh, nkv, hd, rot, rot_at, halves, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_rope_strided_and_large(dtype):
    check_norm_rope(300, 16, 2, 128, 64, None, True, dtype, strided=True)
    check_norm_rope(1100, 24, 24, 64, 64, None, False, dtype)   # many tokens: several heads a group


@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_rope_without_norm_weights_or_rotation(dtype):
    check_norm_rope(4, 6, 2, 128, 64, 0, True, dtype, norm=False, weights=False)
    check_norm_rope(4, 6, 2, 128, 0, None, True, dtype, norm=True, weights=False)
    check_norm_rope(4, 6, 2, 96, 32, None, False, dtype, norm=False)


def test_norm_rope_padding_and_positions_outside_the_table():
    from microkimi_amd import mixer
    torch = torch_cuda()
    rng = np.random.default_rng(4)
    x = to_dev(rows(rng, (4, 2, 64), "f32"))
    x[1] = float("nan")                                     # a padding row may hold anything
    cos, sin = mixer.rope_table(10, 32)
    out = torch.full_like(x, 7.0)
    got, none = mixer.qk_norm_rope(x, None, cos, sin, ints([3, -1, 10, 2147483647]), q_out=out)
    assert none is None and got is out
    assert torch.equal(got[1], torch.full_like(got[1], 7.0))
    assert torch.isfinite(got[0]).all()
    for r in (2, 3):                                         # no such row in the table: the rotated half is NaN, the rest is not
        assert torch.isnan(got[r][:, 32:]).all() and torch.isfinite(got[r][:, :32]).all()


def test_norm_rope_zero_row_infinity_and_in_place():
    from microkimi_amd import mixer
    torch = torch_cuda()
    rng = np.random.default_rng(5)
    a = rows(rng, (3, 2, 128), "f32")
    a[0, 0], a[1, 1, 3] = 0.0, np.inf
    q = to_dev(a)
    cos, sin = mixer.rope_table(8, 64)
    pos = ints([1, 2, 3])
    want, _ = mixer.qk_norm_rope(q, None, cos, sin, pos, halves=True)
    assert float(want[0, 0].abs().max()) == 0.0
    assert torch.isnan(want[1, 1]).any() and torch.isfinite(want[1, 0]).all()
    q2 = q.clone()
    got, _ = mixer.qk_norm_rope(q2, None, cos, sin, pos, halves=True, q_out=q2)
    assert got is q2 and torch.equal(got.nan_to_num(9.0), want.nan_to_num(9.0))
    empty, _ = mixer.qk_norm_rope(q[:0], None, cos, sin, pos[:0])
    assert empty.shape == (0, 2, 128)


# -------------------------------------------------------------------------------------------------------- 4-bit KV cache

def split(rng, lens, shape, dtype):
    return [rows(rng, (n,) + shape, dtype) for n in lens]


def cu_of(lens):
    return ints(np.concatenate([[0], np.cumsum(lens)]))


def held(k, dk, v):
    """The values a cache stands for after k [n, nkv, dk + rope], v [n, nkv, dv] were stored."""
    kk = np.concatenate([ref.mxfp4(k[..., :dk]), np.broadcast_to(ref.bf16(k[:, :1, dk:]), k[..., dk:].shape).astype(np.float64)], -1)
    return kk, ref.mxfp4(v)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nkv,dk,rope,dv", [(3, 128, 64, 128), (8, 128, 0, 128), (1, 32, 8, 512), (2, 256, 0, 64)])
def test_kv4_store_and_snapshot(nkv, dk, rope, dv, dtype):
    from microkimi_amd import mixer
    rng = np.random.default_rng(dk + rope)
    lens1, lens2, cap = [3, 0, 17], [1, 4, 2], 20
    c = mixer.KvCache4(3, nkv, dk, dv, cap, rope=rope)
    ks, vs = [], []
    for lens in (lens1, lens2):
        k, v = split(rng, lens, (nkv, dk + rope), dtype), split(rng, lens, (nkv, dv), dtype)
        if lens is lens2:  # blocks that are zero, tiny, huge, not finite, and one at a midpoint
            k[0][0, 0, :32] = 0.0
            v[0][0, 0, :32] *= 1e-30
            v[2][1, nkv - 1, :32] *= 1e30
            k[1][2, 0, 3:6] = [np.nan, np.inf, -np.inf]
            v[1][0, 0, :4] = [6.0, 2.5, 0.25, -5.0]
            if dtype == "bf16":
                v = [ref.bf16(x) for x in v]
        c.push(to_dev(np.concatenate(k), dtype), to_dev(np.concatenate(v), dtype), cu=cu_of(lens))
        ks.append(k), vs.append(v)
    assert c.positions() == [4, 4, 19]
    gk, gv = c.to_f32()
    assert gk.shape == (3, cap, nkv, dk + rope)
    for b in range(3):
        wk, wv = held(np.concatenate([ks[0][b], ks[1][b]]), dk, np.concatenate([vs[0][b], vs[1][b]]))
        n = wk.shape[0]
        assert np.array_equal(host(gk[b, :n]), wk.astype(np.float32)) and np.array_equal(host(gv[b, :n]), wv.astype(np.float32))
        assert not host(gk[b, n:]).any() and not host(gv[b, n:]).any()
    c.assign(to_dev(ks[0][2], dtype), to_dev(vs[0][2], dtype), cu=ints([0, 0, 17, 17]))
    assert c.positions() == [0, 17, 0]
    gk, gv = c.to_f32(18)
    wk, wv = held(ks[0][2], dk, vs[0][2])
    assert np.array_equal(host(gk[1, :17]), wk.astype(np.float32)) and np.array_equal(host(gv[1, :17]), wv.astype(np.float32))
    assert not host(gk[0]).any() and not host(gk[1, 17]).any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_kv4_levels_at_and_beside_every_midpoint(dtype):
    """Rounding is exact arithmetic: the values held equal the definition's, signs of zeros included."""
    from microkimi_amd import mixer
    mids = np.array([.25, .75, 1.25, 1.75, 2.5, 3.5, 5.0], np.float32)
    near = np.concatenate([mids, mids * np.float32(1 - 2.0 ** -8), mids * np.float32(1 + 2.0 ** -7), np.nextafter(mids, np.float32(0)), np.nextafter(mids, np.float32(9))])
    special = np.array([0.0, -0.0, np.nan, 1e-40, -1e-40, 0.2, -0.2], np.float32)
    vals = np.concatenate([near, -near, special])
    vals = np.concatenate([vals, np.zeros(-len(vals) % 31, np.float32)]).reshape(-1, 31)
    blocks = []
    for top in (6.0, 4.5, 4.0, 3.2):      # a block's largest value sets its exponent
        for ex in (-120, -30, -1, 0, 1, 40, 124):
            b = np.concatenate([np.minimum(np.abs(vals), np.float32(top)) * np.copysign(1, vals), np.full((len(vals), 1), top, np.float32)], 1).astype(np.float32)
            blocks.append(np.ldexp(b, ex).astype(np.float32))
    blocks += [np.where(np.arange(32) % 5 == 0, np.float32(x), b).astype(np.float32) for b in blocks[:2] for x in (np.inf, -np.inf, 3e38, -3e38)]
    x = np.concatenate(blocks)
    if dtype == "bf16":
        x = ref.bf16(x).astype(np.float32)
    n = len(x)
    c = mixer.KvCache4(1, 1, 32, 32, n)
    c.push(to_dev(x[:, None], dtype), to_dev(-x[:, None], dtype))
    k, v = c.to_f32()
    for got, src in ((host(k[0, :, 0]), x), (host(v[0, :, 0]), -x)):
        want = ref.mxfp4(src).astype(np.float32)
        assert np.array_equal(got, want) and np.array_equal(np.signbit(got), np.signbit(want))


def test_kv4_rows_beyond_the_capacity_and_behind_the_last_sequence():
    from microkimi_amd import mixer
    torch = torch_cuda()
    rng = np.random.default_rng(1)
    c = mixer.KvCache4(2, 1, 32, 32, 4)
    before = c.kq.clone()
    k, v = rows(rng, (9, 1, 32), "f32"), rows(rng, (9, 1, 32), "f32")
    c.push(to_dev(k), to_dev(v), cu=ints([1, 3, 7]))    # row 0 and rows 7, 8 belong to nobody
    assert c.positions() == [2, 4]
    gk, _ = c.to_f32()
    assert np.array_equal(host(gk[0, :2, 0]), ref.mxfp4(k[1:3, 0]).astype(np.float32))
    assert np.array_equal(host(gk[1, :, 0]), ref.mxfp4(k[3:7, 0]).astype(np.float32))
    assert torch.equal(c.kq[0, :, 2:], before[0, :, 2:])
    c.push(to_dev(k[:2]), to_dev(v[:2]))                  # one row each; sequence 1 is full
    assert c.positions() == [3, 5]
    gk2, _ = c.to_f32()
    assert torch.equal(gk2[1], gk[1]) and np.array_equal(host(gk2[0, 2, 0]), ref.mxfp4(k[0, 0]).astype(np.float32))
    out = c.attn(to_dev(rows(rng, (2, 2, 32), "f32")), 0.2)
    assert torch.isfinite(out[0]).all() and torch.isnan(out[1]).all()


def check_attn(lens, news, nh, nkv, dk, rope, dv, dtype, seed=0, sharp=1.0, cap=None, uniform=False, strided=False, max_len=None, tail_rows=0, scale=None):
    """Sequences of lens positions, of which the last news[b] are the rows of the call."""
    from microkimi_amd import mixer
    torch = torch_cuda()
    rng = np.random.default_rng(seed)
    B, cap = len(lens), cap or max(max(lens), 1) + 3
    c = mixer.KvCache4(B, nkv, dk, dv, cap, rope=rope)
    for t in (c.kq, c.ks, c.vq, c.vs):
        t.fill_(255)                                          # what lies behind a sequence must not matter: NaN scales
    if rope:
        c.kr.fill_(float("nan"))
    k, v = split(rng, lens, (nkv, dk + rope), dtype), split(rng, lens, (nkv, dv), dtype)
    c.push(to_dev(np.concatenate(k), dtype), to_dev(np.concatenate(v), dtype), cu=cu_of(lens))
    T = sum(news)
    qn = rows(rng, (T, nh, dk + rope), dtype) * np.float32(sharp)
    qn = ref.bf16(qn) if dtype == "bf16" else qn   # (the scaled rows as the device holds them)
    q = to_dev(qn, dtype)
    if tail_rows:
        q = torch.cat((q, torch.full((tail_rows, nh, dk + rope), float("nan"), dtype=q.dtype, device="cuda")))
    if strided:
        wide = torch.full((q.shape[0], nh + 2, dk + rope), float("nan"), dtype=q.dtype, device="cuda")
        wide[:, 1:-1] = q
        q = wide[:, 1:-1]
    out = torch.full((q.shape[0], nh, dv), 7.0, dtype=q.dtype, device="cuda")
    scale = (dk + rope) ** -0.5 if scale is None else scale
    got = host(c.attn(q, scale, cu=None if uniform else cu_of(news), out=out, max_len=max_len))
    assert (got[T:] == 7.0).all()
    t, wants = 0, []
    for b in range(B):
        kk, vv = held(k[b], dk, v[b])
        for i in range(news[b]):
            want, bound, mag = ref.attn(qn[t], kk, vv, lens[b] - news[b] + i, scale)
            # bfloat16 rows: the weights may enter the product with V rounded to bfloat16, and so does the result
            tol = bound * U32 + (U16 * mag + U16 * (np.abs(want) + U16 * mag) if dtype == "bf16" else 0)
            within(got[t], want, tol + 1e-30, f"sequence {b} row {i}")
            wants.append(want)
            t += 1
    if T and np.abs(np.stack(wants)).max() > 0:
        assert rel_l2(got[:T], np.stack(wants)) <= (1e-5 if dtype == "f32" else 2 * U16)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nh,nkv,dk,rope,dv", [(3, 3, 128, 64, 128), (16, 2, 128, 0, 128), (40, 8, 64, 0, 64), (5, 1, 256, 0, 256), (34, 2, 128, 64, 128),
                                               (4, 2, 96, 8, 160), (20, 1, 64, 64, 64)])
@pytest.mark.parametrize("lens", [[1], [2, 0, 33], [300, 31, 1, 64, 129]])
def test_kv4_decode(lens, nh, nkv, dk, rope, dv, dtype):
    check_attn(lens, [1] * len(lens), nh, nkv, dk, rope, dv, dtype, seed=len(lens), uniform=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nh,nkv,dk,rope,dv", [(2, 2, 128, 64, 128), (16, 2, 128, 0, 128), (4, 1, 64, 0, 64), (3, 3, 256, 0, 256), (4, 2, 96, 8, 160)])
def test_kv4_prompt(nh, nkv, dk, rope, dv, dtype):
    check_attn([37, 5, 130], [37, 0, 70], nh, nkv, dk, rope, dv, dtype, seed=3, tail_rows=2)
    check_attn([3, 40], [3, 19], nh, nkv, dk, rope, dv, dtype, seed=4, strided=True)


@pytest.mark.parametrize("dtype", DTYPES)
def test_kv4_long_contexts(dtype):
    check_attn([5003], [1], 4, 2, 128, 64, 128, dtype, seed=6, uniform=True, cap=8192)
    check_attn([3000, 1], [2, 1], 8, 1, 128, 0, 128, dtype, seed=7, max_len=3000)
    check_attn([2100], [9], 16, 2, 64, 0, 64, dtype, seed=8)


@pytest.mark.parametrize("dtype", DTYPES)
def test_kv4_many_sequences_of_every_length(dtype):
    lens = [[0, 1, 40, 1030, 7, 0, 300][i % 7] for i in range(69)] + [2590]
    check_attn(lens, [min(n, 1) for n in lens], 4, 2, 64, 0, 64, dtype, seed=12)
    check_attn(lens, [1] * 70, 2, 2, 64, 64, 64, dtype, seed=13, uniform=True, max_len=1500)   # (a hint that is too small)
    check_attn([1300, 0, 1100, 64], [70, 0, 3, 64], 2, 2, 128, 0, 128, dtype, seed=14, cap=4096)


@pytest.mark.parametrize("dtype", DTYPES)
def test_kv4_prompts_in_pieces_and_uncut(dtype):
    check_attn([1500, 40], [20, 3], 16, 2, 256, 0, 256, dtype, seed=15)
    check_attn([1100], [33], 2, 2, 256, 64, 256, dtype, seed=16)
    check_attn([1300], [300], 4, 2, 96, 8, 160, dtype, seed=17)      # widths without a matrix kernel: 1200 workgroups, no pieces
    check_attn([9, 20, 1], [9, 2, 1], 8, 2, 128, 64, 128, dtype, seed=18, cap=20)   # fewer than 32 positions of room


@pytest.mark.parametrize("dtype", DTYPES)
def test_kv4_sharp_scores(dtype):
    check_attn([700], [1], 4, 2, 128, 0, 128, dtype, seed=9, sharp=30.0, uniform=True)
    check_attn([90], [33], 4, 2, 128, 64, 128, dtype, seed=10, sharp=30.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nh,nkv,dk,rows_", [(4, 2, 128, 1), (4, 2, 64, 40), (2, 1, 96, 5)])
@pytest.mark.parametrize("scale", [0.0, -0.0, -0.3, 1e-42])
def test_kv4_scales_that_are_zero_negative_or_tiny(nh, nkv, dk, rows_, scale, dtype):
    check_attn([50, 41], [rows_, rows_], nh, nkv, dk, 0, dk, dtype, seed=19, scale=scale)


@pytest.mark.parametrize("dtype", DTYPES)
def test_kv4_a_query_that_is_not_finite_stays_in_its_row(dtype):
    from microkimi_amd import mixer
    torch = torch_cuda()
    rng = np.random.default_rng(2)
    c = mixer.KvCache4(1, 2, 128, 128, 64)
    k, v, q = (to_dev(rows(rng, s, dtype), dtype) for s in ((40, 2, 128), (40, 2, 128), (20, 4, 128)))
    v[39, 0, 5], k[38, 1, 7] = float("inf"), float("nan")    # held as finite values: no earlier row is touched either
    c.push(k, v)
    want = c.attn(q, 0.1)
    assert torch.isfinite(want).all()
    q[3, 1, 0], q[7, 2, 5] = float("nan"), float("inf")
    got = c.attn(q, 0.1)
    hit = torch.zeros((20, 4), dtype=torch.bool, device="cuda")
    hit[3, 1] = hit[7, 2] = True
    assert torch.equal(got[~hit], want[~hit])
    assert torch.isnan(got[3, 1]).all() and torch.isnan(got[7, 2]).all()


# ------------------------------------------------------------------------------------------------------ linear attention

def check_linear(lens, nh, nkh, dk, dv, dtype, seed=0, per_token=True, with_state=True, tail_rows=0, strided=False, step=False, resets=False, speed=0.2):
    from microkimi_amd import mixer
    torch = torch_cuda()
    rng = np.random.default_rng(seed)
    B, T = len(lens), sum(lens)
    q, k, v = rows(rng, (T, nkh, dk), dtype), rows(rng, (T, nkh, dk), dtype), rows(rng, (T, nh, dv), dtype)
    g = -(speed * rng.random((T, nh) if per_token else nh)).astype(np.float32)
    if resets and T > 2:
        g[rng.integers(0, T, max(1, T // 40))] = -np.inf
        g[rng.integers(0, T, max(1, T // 60)), 0] = -150.0
    state = rng.standard_normal((B, nh, dk, dv)).astype(np.float32) if with_state else None
    scale = dk ** -0.5
    tq, tk, tv, tg = to_dev(q, dtype), to_dev(k, dtype), to_dev(v, dtype), to_dev(g)
    if tail_rows:
        pad = lambda t: torch.cat((t, torch.full((tail_rows,) + tuple(t.shape[1:]), float("nan"), dtype=t.dtype, device="cuda")))
        tq, tk, tv = pad(tq), pad(tk), pad(tv)
        tg = pad(tg) if per_token else tg
    if strided:
        def inside(t):
            w = torch.full((t.shape[0], t.shape[1] + 2, t.shape[2]), float("nan"), dtype=t.dtype, device="cuda")
            w[:, 1:-1] = t
            return w[:, 1:-1]
        tq, tk, tv = inside(tq), inside(tk), inside(tv)
    out = torch.full((T + tail_rows, nh, dv), 7.0, dtype=tv.dtype, device="cuda")
    ts = to_dev(state) if with_state else None
    keep = ts.clone() if with_state else None
    if step:
        got, new = mixer.linear_attn_step(tq, tk, tv, tg, ts, scale, out=out)
    else:
        got, new = mixer.linear_attn(tq, tk, tv, tg, ts, scale, cu=cu_of(lens), out=out)
    if with_state:
        assert torch.equal(ts, keep)
        new2 = ts.clone()
        if not step:                                            # in place: the same state
            mixer.linear_attn(tq, tk, tv, tg, new2, scale, cu=cu_of(lens), state_out=new2)
            assert torch.equal(new2, new)
    assert got is out
    got, new, t = host(got), host(new), 0
    assert (got[T:] == 7.0).all()
    for b, n in enumerate(lens):
        gb = g[t:t + n] if per_token else np.broadcast_to(g, (n, nh))
        s0 = state[b] if with_state else np.zeros((nh, dk, dv), np.float32)
        want, S, mag, M = ref.linear(q[t:t + n], k[t:t + n], v[t:t + n], gb, s0, scale)
        # a chain of n decays and additions and, per output, sums of dk and n products: one half step of the magnitude each, and 24
        # for the exponentials and the products.  bfloat16 rows: inside a block the weighted scores, behind it the state may enter
        # their products rounded to bfloat16 (either, for a term of the output), and the result is rounded
        f32 = (2 * n + dk + 24) * U32
        tol = f32 * mag + (U16 * mag + U16 * (np.abs(want) + U16 * mag) if dtype == "bf16" else 0)
        within(got[t:t + n], want, tol + 1e-30, f"out of sequence {b}")
        within(new[b], S, f32 * M + 1e-30, f"state of sequence {b}")
        assert rel_l2(new[b], S) <= 1e-6 * max(1.0, (n / 1000) ** 0.5)
        # in all: 1e-5 (bfloat16: two roundings) of the result, plus one rounding of each of a dot product's dk terms, which a
        # result that has cancelled does not cover (one token, no state: out = scale (q . k) v, and q . k may be anything)
        err = np.linalg.norm(got[t:t + n] - want)
        assert err <= (1e-5 if dtype == "f32" else 2 * U16) * np.linalg.norm(want) + (dk + 24) * U32 * np.linalg.norm(mag)
        t += n


SHAPES = [(2, 2, 128, 128), (4, 2, 64, 128), (3, 1, 128, 64), (2, 2, 64, 64), (2, 1, 40, 72), (1, 1, 256, 256), (2, 2, 8, 8)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nh,nkh,dk,dv", SHAPES)
def test_linear_prompts(nh, nkh, dk, dv, dtype):
    check_linear([70, 0, 1, 64, 129], nh, nkh, dk, dv, dtype, seed=dk, tail_rows=3)
    check_linear([63, 2], nh, nkh, dk, dv, dtype, seed=dv, per_token=False, strided=True)
    check_linear([33], nh, nkh, dk, dv, dtype, seed=1, with_state=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nh,nkh,dk,dv", SHAPES)
def test_linear_single_tokens(nh, nkh, dk, dv, dtype):
    check_linear([1] * 5, nh, nkh, dk, dv, dtype, seed=2, step=True)
    check_linear([1] * 2, nh, nkh, dk, dv, dtype, seed=3, step=True, per_token=False, with_state=False, strided=True)


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_long_prompts_and_decays(dtype):
    check_linear([1500], 2, 2, 128, 128, dtype, seed=5, speed=0.02)
    check_linear([700, 300], 2, 1, 64, 128, dtype, seed=6, speed=8.0)
    check_linear([400, 100], 2, 2, 128, 128, dtype, seed=7, resets=True)
    check_linear([200], 2, 2, 64, 64, dtype, seed=8, speed=0.0)     # no decay at all


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens", [[0, 300, 1, 1000, 257, 0], [1279, 1], [128, 1664, 128, 0, 0], [5, 2000, 3, 173, 2]])
def test_linear_long_and_short_prompts_side_by_side(lens, dtype):
    check_linear(lens, 2, 1, 64, 64, dtype, seed=len(lens), tail_rows=2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 64), (40, 72)])
def test_linear_values_that_are_not_finite_reach_later_tokens_only(dk, dv, dtype):
    from microkimi_amd import mixer
    torch = torch_cuda()
    rng = np.random.default_rng(11)
    T, nh = 150, 2
    q, k, v = (to_dev(rows(rng, (T, nh, d), dtype), dtype) for d in (dk, dk, dv))
    g = to_dev(-0.1 * rng.random((T, nh)).astype(np.float32))
    want, _ = mixer.linear_attn(q, k, v, g)
    for bad in (float("nan"), float("inf")):
        v2, k2 = v.clone(), k.clone()
        v2[90, 0, 5] = bad
        got, S = mixer.linear_attn(q, k, v2, g)
        assert torch.equal(got[:90], want[:90]) or rel_l2(host(got[:90]), host(want[:90])) <= (1e-5 if dtype == "f32" else 2 * U16)
        assert not torch.isfinite(got[90:, 0, 5]).any() and not torch.isfinite(S[0, 0, :, 5]).any()
        other = torch.ones(dv, dtype=torch.bool, device="cuda")
        other[5] = False
        assert rel_l2(host(got[:, :, other]), host(want[:, :, other])) <= (1e-5 if dtype == "f32" else 2 * U16)
        k2[90, 1, 3] = bad
        got, S = mixer.linear_attn(q, k2, v, g)
        assert torch.isfinite(got[:90]).all() and torch.isfinite(got[:, 0]).all() and not torch.isfinite(got[90:, 1]).any()
        g2 = g.clone()
        g2[120:] = float("-inf")                                # e^-inf = 0 empties the state, but 0 * inf stays NaN
        got, _ = mixer.linear_attn(q, k, v2, g2)
        assert torch.isfinite(got[:90]).all() and torch.isnan(got[120:, 0, 5]).all()


# -------------------------------------------------------------------------------------------------------------- together

def layer(mixer, cache, state, q, k, v, ql, kl, vl, g, table, pos, cu):
    """One softmax-attention and one linear-attention mixer on the same tokens, as two layers of a hybrid model run them."""
    q, k = mixer.qk_norm_rope(q, k, *table, pos, halves=True)
    cache.push(k, v, cu=cu)
    a = cache.attn(q, 128 ** -0.5, cu=cu)
    ql, kl = mixer.qk_norm_rope(ql, kl, *table, pos, halves=True)
    o, _ = mixer.linear_attn(ql, kl, vl, g, state, 128 ** -0.5, cu=cu, state_out=state) if cu is not None else \
        mixer.linear_attn_step(ql, kl, vl, g, state, 128 ** -0.5, state_out=state)
    return a, o


def make_tokens(rng, T, dtype):
    return [to_dev(rows(rng, (T, h, 128), dtype), dtype) for h in (16, 2, 2, 4, 4, 4)] + [to_dev(-0.1 * rng.random((T, 4)).astype(np.float32))]


@pytest.mark.parametrize("dtype", DTYPES)
def test_prompt_then_tokens_equal_the_prompt_at_once(dtype):
    # prompts of three sequences and then four single tokens each, against one call over all tokens
    from microkimi_amd import mixer
    torch = torch_cuda()
    rng = np.random.default_rng(21)
    lens, extra = [70, 1, 33], 4
    table = mixer.rope_table(256, 128)
    full = [n + extra for n in lens]
    tok = make_tokens(rng, sum(full), dtype)
    starts = np.concatenate([[0], np.cumsum(full)])
    new = lambda: (mixer.KvCache4(3, 2, 128, 128, 128), torch.zeros((3, 4, 128, 128), device="cuda"))
    cache, state = new()
    pos_all = ints(np.concatenate([np.arange(n) for n in full]))
    want_a, want_o = layer(mixer, cache, state, *tok, table, pos_all, cu_of(full))
    cache2, state2 = new()
    take = lambda idx: [t[idx] for t in tok]
    prompt = torch.from_numpy(np.concatenate([np.arange(s, s + n) for s, n in zip(starts, lens)])).cuda()
    got_a, got_o = torch.empty_like(want_a), torch.empty_like(want_o)
    got_a[prompt], got_o[prompt] = layer(mixer, cache2, state2, *take(prompt), table, pos_all[prompt], cu_of(lens))
    for i in range(extra):
        idx = torch.tensor([s + n + i for s, n in zip(starts, lens)], device="cuda")
        got_a[idx], got_o[idx] = layer(mixer, cache2, state2, *take(idx), table, pos_all[idx], None)
    assert cache2.positions() == full
    assert torch.equal(cache.kq, cache2.kq) and torch.equal(cache.vs, cache2.vs)
    tol = 1e-5 if dtype == "f32" else 2 * U16 * 2   # two evaluations
    assert rel_l2(host(got_a), host(want_a)) <= tol and rel_l2(host(got_o), host(want_o)) <= tol
    assert rel_l2(host(state2), host(state)) <= 2e-6


@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_step_captured_and_replayed(dtype):
    # one graph of a decode step, replayed with the eager step of a twin between the replays
    from microkimi_amd import mixer
    torch = torch_cuda()
    rng = np.random.default_rng(22)
    table = mixer.rope_table(256, 128)
    mk = lambda: (mixer.KvCache4(2, 2, 128, 128, 64), torch.zeros((2, 4, 128, 128), device="cuda"))
    (c1, s1), (c2, s2) = mk(), mk()
    buf, pos = make_tokens(rng, 2, dtype), ints([0, 0])
    layer(mixer, *mk(), *buf, table, pos, None)     # everything loaded before the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, o = layer(mixer, c1, s1, *buf, table, pos, None)
    for step in range(5):
        tok = make_tokens(rng, 2, dtype)
        for t, n in zip(buf, tok):
            t.copy_(n)
        pos.fill_(step)
        graph.replay()
        wa, wo = layer(mixer, c2, s2, *tok, table, ints([step, step]), None)
        torch.cuda.synchronize()
        assert torch.equal(a, wa) and torch.equal(o, wo) and torch.equal(s1, s2) and c1.positions() == c2.positions() == [step + 1] * 2


def test_calls_on_two_streams_at_once():
    from microkimi_amd import mixer
    torch = torch_cuda()
    rng = np.random.default_rng(23)
    c = mixer.KvCache4(1, 8, 128, 128, 4096)
    c.push(*(to_dev(rows(rng, (4000, 8, 128), "bf16"), "bf16") for _ in range(2)))
    qs = [to_dev(rows(rng, (1, 64, 128), "bf16"), "bf16") for _ in range(2)]
    lin = [[to_dev(rows(rng, (600, 4, 128), "bf16"), "bf16") for _ in range(3)] + [to_dev(-0.1 * rng.random((600, 4)).astype(np.float32))] for _ in range(2)]
    want = [(c.attn(q, 0.1), *mixer.linear_attn(*x)) for q, x in zip(qs, lin)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append((c.attn(qs[i], 0.1), *mixer.linear_attn(*lin[i])))
    torch.cuda.synchronize()
    for i in range(2):
        for triple in got[i]:
            assert all(torch.equal(x, y) for x, y in zip(triple, want[i]))


def test_a_call_without_sequences_is_refused():
    from microkimi_amd import mixer
    torch = torch_cuda()
    x, g = torch.zeros((4, 2, 64), device="cuda"), torch.zeros((4, 2), device="cuda")
    for kw in (dict(B=0), dict(B=-1), dict(cu=ints([0]))):
        with pytest.raises(ValueError, match="sequence"):
            mixer.linear_attn(x, x, x, g, **kw)
    with pytest.raises(ValueError):
        mixer.KvCache4(0, 1, 32, 32, 4)


# ------------------------------------------------------------------------------------------- offsets that pass 32 bits

def test_norm_rope_beyond_four_gigabytes():
    from microkimi_amd import mixer
    torch = torch_cuda()
    T, nh = 2 ** 18 + 3, 64
    q = torch.empty((T, nh, 128), dtype=torch.bfloat16, device="cuda").normal_()     # 2^31 values and some
    k = torch.empty((T, 1, 128), dtype=torch.bfloat16, device="cuda").normal_()
    cos, sin = mixer.rope_table(4096, 64)
    pos = torch.arange(T, dtype=torch.int32, device="cuda") % 4096
    qo, ko = mixer.qk_norm_rope(q, k, cos, sin, pos, halves=True)
    for a, b in ((0, 3), (T // 2, T // 2 + 2), (T - 3, T)):
        wq, wk = mixer.qk_norm_rope(q[a:b], k[a:b], cos, sin, pos[a:b], halves=True)
        assert torch.equal(qo[a:b], wq) and torch.equal(ko[a:b], wk)
    del q, k, qo, ko
    torch.cuda.empty_cache()


@pytest.mark.parametrize("new", [1, 40])
def test_kv4_cache_beyond_four_gigabytes(new):
    """A cache at its largest capacity, zeros but for the last rows, whose scores stand far above: the last head's K and V lie
    behind the 4 GiB of the others."""
    from microkimi_amd import mixer
    torch = torch_cuda()
    rng = np.random.default_rng(5)
    nkv, cap = 9, 8388607
    c = mixer.KvCache4(1, nkv, 128, 128, cap, rope=64)
    assert c.kq.numel() > 2 ** 32
    c.lens.fill_(cap - new)
    k, v = rows(rng, (new, nkv, 192), "f32"), rows(rng, (new, nkv, 128), "f32")
    c.push(to_dev(k), to_dev(v))
    kk, vv = held(k, 128, v)
    q = np.repeat(kk[:1].astype(np.float32), new, 0)          # the first new row's own K: |k|^2 against a few |k| elsewhere
    scale = 40.0 / float((kk[0] ** 2).sum(-1).min())
    out = host(c.attn(to_dev(q), scale))
    for i in range(new):
        s = np.einsum("hw,jhw->jh", q[i].astype(np.float64), kk[:i + 1]) * scale
        p = np.exp(s)
        den = p.sum(0) + (cap - new)
        want, mag = np.einsum("jh,jhd->hd", p, vv[:i + 1]) / den[:, None], np.einsum("jh,jhd->hd", p, np.abs(vv[:i + 1])) / den[:, None]
        # as in mixer_ref.attn for the rows that count; the zeros' share of the sum is below 8.4e6 e^-40 = 4e-11
        ds = 194 * (np.abs(q[i].astype(np.float64)) * np.abs(kk[:i + 1])).sum(-1).max() * scale
        within(out[i], want, (2 * ds + new + 16) * mag * U32 + 1e-30, f"row {i}")
    del c
    torch.cuda.empty_cache()


def test_linear_beyond_four_gigabytes():
    from microkimi_amd import mixer
    torch = torch_cuda()
    T, nh = 2 ** 19 + 100, 32
    q = torch.empty((T, 1, 64), dtype=torch.bfloat16, device="cuda").normal_()
    k = torch.empty((T, 1, 64), dtype=torch.bfloat16, device="cuda").normal_()
    v = torch.empty((T, nh, 128), dtype=torch.bfloat16, device="cuda").normal_()      # 2^31 values and some
    g = torch.full((nh,), -0.5, device="cuda")
    out, S = mixer.linear_attn(q, k, v, g)
    for end in (T, T // 2):                                     # e^-220 of what lies 440 tokens back: nothing
        want, W = mixer.linear_attn(q[end - 704:end], k[end - 704:end], v[end - 704:end], g)
        assert rel_l2(host(out[end - 256:end]), host(want[-256:])) <= 4 * U16
    want, W = mixer.linear_attn(q[-704:], k[-704:], v[-704:], g)
    assert rel_l2(host(S), host(W)) <= 1e-5
    del q, k, v, out
    torch.cuda.empty_cache()


# --------------------------------------------------------------------------------------- bfloat16 results are rounded once

def rounded_once(got, want, before, what):
    """got is a value within `before` of want, rounded to bfloat16."""
    within(got, want, before + U16 * (np.abs(want) + before) + 1e-30, what)


@pytest.mark.parametrize("lens,news,nh,nkv,dk,rope", [([700, 90], [90, 33], 4, 2, 128, 64), ([1200], [200], 8, 1, 64, 0), ([300, 40], [1, 1], 40, 2, 128, 0),
                                                      ([20, 9], [1, 9], 4, 2, 64, 64), ([260], [70], 2, 2, 256, 0), ([900, 7], [1, 1], 6, 2, 128, 0)])
def test_kv4_a_bfloat16_result_is_rounded_once(lens, news, nh, nkv, dk, rope):
    """Prompts, wide groups, small caches and plain decoding.  A weight may enter its product as two bfloat16 terms: what is left of it is
    half a step of half a step, U16^2."""
    from microkimi_amd import mixer
    rng = np.random.default_rng(31 + sum(lens))
    c = mixer.KvCache4(len(lens), nkv, dk, dk, max(lens), rope=rope)
    k, v = split(rng, lens, (nkv, dk + rope), "bf16"), split(rng, lens, (nkv, dk), "bf16")
    c.push(to_dev(np.concatenate(k), "bf16"), to_dev(np.concatenate(v), "bf16"), cu=cu_of(lens))
    q = rows(rng, (sum(news), nh, dk + rope), "bf16")
    scale = (dk + rope) ** -0.5
    got, t = host(c.attn(to_dev(q, "bf16"), scale, cu=cu_of(news))), 0
    for b in range(len(lens)):
        kk, vv = held(k[b], dk, v[b])
        for i in range(news[b]):
            want, bound, mag = ref.attn(q[t], kk, vv, lens[b] - news[b] + i, scale)
            rounded_once(got[t], want, bound * U32 + U16 ** 2 * mag, f"sequence {b} row {i}")
            t += 1


@pytest.mark.parametrize("nh,nkh,dk,dv", [(2, 2, 128, 128), (4, 2, 64, 128), (3, 1, 128, 64), (2, 2, 64, 64), (2, 1, 40, 72)])
@pytest.mark.parametrize("lens,with_state", [([70, 0, 1, 64, 129], True), ([1000], True), ([100], False), ([900, 3, 300], True)])
def test_linear_a_bfloat16_result_is_rounded_once(lens, with_state, nh, nkh, dk, dv):
    """One workgroup a sequence, and segments.  The state and the weighted scores may enter their products, and where a state only leads to
    later outputs its updates too, as two bfloat16 terms: twice U16^2."""
    from microkimi_amd import mixer
    rng = np.random.default_rng(41 + sum(lens) + dk)
    B, T = len(lens), sum(lens)
    q, k, v = rows(rng, (T, nkh, dk), "bf16"), rows(rng, (T, nkh, dk), "bf16"), rows(rng, (T, nh, dv), "bf16")
    g = -(0.2 * rng.random((T, nh))).astype(np.float32)
    state = rng.standard_normal((B, nh, dk, dv)).astype(np.float32) if with_state else np.zeros((B, nh, dk, dv), np.float32)
    scale = dk ** -0.5
    got, _ = mixer.linear_attn(*(to_dev(x, "bf16") for x in (q, k, v)), to_dev(g), to_dev(state) if with_state else None, scale, cu=cu_of(lens))
    got, t = host(got), 0
    for b, n in enumerate(lens):
        want, _, mag, _ = ref.linear(q[t:t + n], k[t:t + n], v[t:t + n], g[t:t + n], state[b], scale)
        rounded_once(got[t:t + n], want, ((2 * n + dk + 24) * U32 + 2 * U16 ** 2) * mag, f"sequence {b}")
        t += n


# ------------------------------------------------------------------------------------------- rows before the first sequence

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nh,nkh,dk,dv", [(2, 1, 64, 64), (2, 2, 128, 128), (4, 2, 64, 128)])
@pytest.mark.parametrize("cu,T", [([200, 1000], 1000), ([300, 700, 1500], 1600), ([513, 513, 1900, 1901], 1901), ([-7, 90, 5000], 1200)])
def test_linear_rows_before_the_first_sequence_belong_to_nobody(cu, T, nh, nkh, dk, dv, dtype):
    """Long enough for segments: every segment is computed once, from the state before it.  Entries outside 0 .. T count as the nearer bound."""
    from microkimi_amd import mixer
    torch = torch_cuda()
    rng = np.random.default_rng(51 + T)
    B, at = len(cu) - 1, np.clip(cu, 0, T)
    q, k, v = rows(rng, (T, nkh, dk), dtype), rows(rng, (T, nkh, dk), dtype), rows(rng, (T, nh, dv), dtype)
    g = -(0.1 * rng.random((T, nh))).astype(np.float32)
    for a in (q, k, v, g):
        a[:at[0]], a[at[-1]:] = np.nan, np.nan
    state = rng.standard_normal((B, nh, dk, dv)).astype(np.float32)
    out = torch.full((T, nh, dv), 7.0, dtype=to_dev(v[:1], dtype).dtype, device="cuda")
    scale = dk ** -0.5
    got, new = mixer.linear_attn(*(to_dev(x, dtype) for x in (q, k, v)), to_dev(g), to_dev(state), scale, cu=ints(cu), out=out)
    got, new = host(got), host(new)
    assert (got[:at[0]] == 7.0).all() and (got[at[-1]:] == 7.0).all()
    for b in range(B):
        s = slice(at[b], at[b + 1])
        want, S, mag, M = ref.linear(q[s], k[s], v[s], g[s], state[b], scale)
        f32 = (2 * len(want) + dk + 24) * U32      # (as in check_linear; bfloat16: two-term operands, twice U16^2)
        if dtype == "bf16":
            rounded_once(got[s], want, (f32 + 2 * U16 ** 2) * mag, f"sequence {b}")
        else:
            within(got[s], want, f32 * mag + 1e-30, f"sequence {b}")
        within(new[b], S, f32 * M + 1e-30, f"state of sequence {b}")


@pytest.mark.parametrize("T,B,nh,dk,dv", [(512, 1, 160, 64, 128), (1280, 2, 65, 128, 128), (300, 1, 191, 128, 64)])
def test_linear_equal_f32_sequences_are_not_cut_into_one_segment_each(T, B, nh, dk, dv):
    """A segment a sequence is the same workgroups three times over: such calls leave their workspace alone."""
    from microkimi_amd._lib import F32, check, lib
    torch = torch_cuda()
    rng = np.random.default_rng(61)
    q, k, v = (rng.standard_normal((T, h, w)).astype(np.float32) for h, w in ((1, dk), (1, dk), (nh, dv)))
    g = -(0.1 * rng.random((T, nh))).astype(np.float32)
    tq, tk, tv, tg = to_dev(q), to_dev(k), to_dev(v), to_dev(g)
    n = lib.mk_linear_attn_workspace_bytes(T, B, nh, dk, dv)
    ws = torch.full((n,), 77, dtype=torch.uint8, device="cuda")
    out, S = torch.empty((T, nh, dv), device="cuda"), torch.empty((B, nh, dk, dv), device="cuda")
    check(lib.mk_dev_linear_attn(F32, tq.data_ptr(), dk, tk.data_ptr(), dk, tv.data_ptr(), nh * dv, tg.data_ptr(), nh, T, None, B, nh, 1, dk, dv, 0.1, None,
                                 S.data_ptr(), ws.data_ptr(), out.data_ptr(), torch.cuda.current_stream().cuda_stream))
    assert (ws == 77).all()
    out, S, m = host(out), host(S), T // B
    for b in range(B):
        s, h = slice(b * m, (b + 1) * m), [0, 1, nh // 2, nh - 1]
        want, W, mag, M = ref.linear(np.repeat(q[s], 4, 1), np.repeat(k[s], 4, 1), v[s][:, h], g[s][:, h], np.zeros((4, dk, dv), np.float32), 0.1)
        f32 = (2 * m + dk + 24) * U32
        within(out[s][:, h], want, f32 * mag + 1e-30, f"sequence {b}")
        within(S[b][h], W, f32 * M + 1e-30, f"state of sequence {b}")


def test_calls_by_torchs_public_stream_and_device(monkeypatch):
    """What mixer uses where torch has no internal forms of them, under a stream of its own."""
    from microkimi_amd import mixer
    torch = torch_cuda()
    x = to_dev(rows(np.random.default_rng(71), (3, 2, 64), "f32"))
    want, _ = mixer.qk_norm_rope(x, None)
    torch.cuda.synchronize()
    with monkeypatch.context() as m:
        m.setattr(mixer, "_current_device", torch.cuda.current_device)
        m.setattr(mixer, "_raw_stream", lambda dev: torch.cuda.current_stream(dev).cuda_stream)
        with torch.cuda.stream(torch.cuda.Stream()):
            got, _ = mixer.qk_norm_rope(x, None)
        torch.cuda.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dk,dv", [(64, 128), (40, 72)])
@pytest.mark.parametrize("per_token", [True, False])
def test_linear_calls_without_a_token(dk, dv, per_token, dtype):
    """No tokens: nothing comes out and every state stays as it is; no sequences of one token: nothing at all."""
    from microkimi_amd import mixer
    torch = torch_cuda()
    q, v = to_dev(np.zeros((0, 2, dk)), dtype), to_dev(np.zeros((0, 4, dv)), dtype)
    g = torch.zeros((0, 4) if per_token else 4, device="cuda")
    S = to_dev(np.random.default_rng(81).standard_normal((3, 4, dk, dv)))
    for cu in (None, ints([0, 0, 0, 0])):
        out, new = mixer.linear_attn(q, q, v, g, S, cu=cu)
        assert out.shape == (0, 4, dv) and torch.equal(new, S)
        out, new = mixer.linear_attn(q, q, v, g, B=2)
        assert out.shape == (0, 4, dv) and new.shape == (2, 4, dk, dv) and not new.any()
    out, new = mixer.linear_attn_step(q, q, v, g)
    assert out.shape == (0, 4, dv) and out.dtype == v.dtype and new.shape == (0, 4, dk, dv)
    mine = torch.empty((0, 4, dv), dtype=v.dtype, device="cuda")
    out, new = mixer.linear_attn_step(q, q, v, g, S[:0], out=mine)
    assert out is mine and new.shape == (0, 4, dk, dv)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 64), (64, 128), (128, 64)])
@pytest.mark.parametrize("at", [0, 127, 128, 255, 300, 699])
def test_linear_values_that_are_not_finite_in_long_prompts(at, dk, dv, dtype):
    """700 tokens are segments of 128: the value stands at a segment's first or last token, inside one, or at the prompt's ends, goes
    through the states of the segments behind it and touches nothing else."""
    from microkimi_amd import mixer
    torch = torch_cuda()
    rng = np.random.default_rng(91)
    T, nh = 700, 2
    q, k, v = (to_dev(rows(rng, (T, nh, d), dtype), dtype) for d in (dk, dk, dv))
    g = to_dev(-0.01 * rng.random((T, nh)).astype(np.float32))
    want, W = mixer.linear_attn(q, k, v, g)
    # the slower sum of a block with such a value and the matrix cores' differ in f32 only: before a bfloat16 rounding (once each)
    tol = 1e-5 if dtype == "f32" else 2 * U16
    column, row = torch.arange(dv, device="cuda") == 5, torch.arange(dk, device="cuda") == 3
    for bad in (float("nan"), float("inf"), float("-inf")):
        v2 = v.clone()
        v2[at, 0, 5] = bad
        got, S = mixer.linear_attn(q, k, v2, g)
        assert not torch.isfinite(got[at:, 0, 5]).any() and not torch.isfinite(S[0, 0, :, 5]).any()
        assert at == 0 or rel_l2(host(got[:at]), host(want[:at])) <= tol
        assert rel_l2(host(got[:, 1]), host(want[:, 1])) <= tol and rel_l2(host(got[..., ~column]), host(want[..., ~column])) <= tol
        assert torch.equal(S[..., ~column], W[..., ~column]) and torch.equal(S[:, 1], W[:, 1])
        k2 = k.clone()
        k2[at, 1, 3] = bad
        got, S = mixer.linear_attn(q, k2, v, g)
        assert not torch.isfinite(got[at:, 1]).any() and not torch.isfinite(S[0, 1, 3]).any()
        assert torch.equal(got[:at], want[:at]) and torch.equal(got[:, 0], want[:, 0])
        assert torch.equal(S[:, 0], W[:, 0]) and torch.equal(S[0, 1, ~row], W[0, 1, ~row])
        q2 = q.clone()
        q2[at, 0, 1] = bad
        got, S = mixer.linear_attn(q2, k, v, g)
        rest = torch.arange(T, device="cuda") != at
        assert torch.equal(got[rest], want[rest]) and torch.equal(got[:, 1], want[:, 1]) and torch.equal(S, W)
        assert not torch.isfinite(got[at, 0]).any()


def test_outputs_that_overlap_what_a_call_still_reads_are_refused():
    """Two workgroups that share a head's columns read all of its query: a result in the same place would overwrite it under the other."""
    from microkimi_amd import mixer
    torch = torch_cuda()
    T, h, d = 3, 2, 128
    q, k, v = (torch.zeros((T, h, d), device="cuda") for _ in range(3))
    g, pool = torch.zeros(h, device="cuda"), torch.zeros((T + 1, h, d, d), device="cuda")
    for call, S, S1 in ((mixer.linear_attn, pool[:1], pool[1:2]), (mixer.linear_attn_step, pool[:T], None)):
        for x in (q, k):
            with pytest.raises(ValueError, match="overlap"):
                call(q, k, v, g, S, out=x)
        if S1 is not None:
            out, new = call(q, k, v, g, S, out=torch.empty_like(v), state_out=S1)     # side by side is not an overlap
            assert new is S1
        out, new = call(q, k, v, g, S, state_out=S)
        assert new is S
    row = torch.zeros((1, 4 * h, d), device="cuda")                                     # one token: slices of one row
    out, _ = mixer.linear_attn_step(row[:, :h], row[:, h:2 * h], row[:, 2 * h:3 * h], g, out=row[:, 3 * h:])
    assert out.data_ptr() == row[:, 3 * h:].data_ptr()
    fused = torch.zeros((T, 3 * h, d), device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        mixer.linear_attn(fused[:, :h], fused[:, h:2 * h], fused[:, 2 * h:], g, out=fused.view(-1)[:T * h * d].view(T, h, d))
    with pytest.raises(ValueError, match="overlap"):
        mixer.qk_norm_rope(q, k, q_out=k)
    with pytest.raises(ValueError, match="overlap"):
        mixer.qk_norm_rope(q, k, k_out=q)
