"""The token-mixer operators as a user's program calls them, with the sizes they are measured at: head norm + rotation,
the 4-bit KV cache (append, snapshot, attention) and linear attention with a decay per head (chunked and one token).

Every case names an operator ("op"), its element type and its sizes.  `run` computes it in plain torch operations, or,
with `own` set, through the framework's entry points; `exact` states the definition once more in 64 bits.
"""
import math
import random

import torch

own = False

F32, BF16 = "f32", "bf16"


def _dt(case):
    return torch.bfloat16 if case["dtype"] == BF16 else torch.float32


def _bytes_of(case):
    return 2 if case["dtype"] == BF16 else 4


# ------------------------------------------------------------------------------------------------------------- the cases

def listed():
    return [
        # one decode token in front of attention with 96 heads of 128 + 64: latency
        {"name": "norm_rope_1x96_f32", "op": "norm_rope", "dtype": F32, "T": 1, "nh": 96, "nkv": 96, "hd": 192, "rot": 64, "halves": False},
        # a prompt of grouped-query heads, the whole head rotated
        {"name": "norm_rope_8192x64_bf16", "op": "norm_rope", "dtype": BF16, "T": 8192, "nh": 64, "nkv": 8, "hd": 128, "rot": 128, "halves": True},
        # an odd chunk of a prompt in the framework's f32
        {"name": "norm_rope_777x96_f32", "op": "norm_rope", "dtype": F32, "T": 777, "nh": 96, "nkv": 96, "hd": 192, "rot": 64, "halves": False},
        # sixteen sequences take their first token
        {"name": "kv4_store_16x1_bf16", "op": "kv4_store", "dtype": BF16, "B": 16, "lo": 1, "hi": 1, "pick": 1, "nkv": 8, "dk": 128, "rope": 0,
         "dv": 128},
        # four prompts of different lengths are stored, and read back as a snapshot
        {"name": "kv4_store_4x2048_bf16", "op": "kv4_store", "dtype": BF16, "B": 4, "lo": 1100, "hi": 2048, "pick": 2, "nkv": 8, "dk": 128, "rope": 0,
         "dv": 128},
        # one decode token behind a short context, the framework's own head shape in f32
        {"name": "kv4_decode_1k_96h_f32", "op": "kv4_attn", "dtype": F32, "B": 1, "lo": 1024, "hi": 1024, "pick": 3, "rows": 1, "nh": 96, "nkv": 96,
         "dk": 128, "rope": 64, "dv": 128},
        # one decode token behind a long context
        {"name": "kv4_decode_16k_96h_bf16", "op": "kv4_attn", "dtype": BF16, "B": 1, "lo": 16384, "hi": 16384, "pick": 4, "rows": 1, "nh": 96,
         "nkv": 96, "dk": 128, "rope": 64, "dv": 128},
        # a serving batch of grouped-query heads, contexts of every length
        {"name": "kv4_decode_32_ragged_gqa_bf16", "op": "kv4_attn", "dtype": BF16, "B": 32, "lo": 1, "hi": 16384, "pick": 5, "rows": 1, "nh": 64,
         "nkv": 8, "dk": 128, "rope": 0, "dv": 128},
        # a prompt chunk of 512 tokens behind 3584 positions
        {"name": "kv4_prompt_512_at_3584_96h_bf16", "op": "kv4_attn", "dtype": BF16, "B": 1, "lo": 4096, "hi": 4096, "pick": 6, "rows": 512,
         "nh": 96, "nkv": 96, "dk": 128, "rope": 64, "dv": 128},
        # one token for each of 64 sequences: the state is read and written once
        {"name": "linear_step_64x32_bf16", "op": "linear_step", "dtype": BF16, "B": 64, "nh": 32, "nkh": 32, "dk": 128, "dv": 128, "per_token": True},
        # a long prompt
        {"name": "linear_8192x32_bf16", "op": "linear", "dtype": BF16, "B": 1, "lo": 8192, "hi": 8192, "pick": 7, "nh": 32, "nkh": 32, "dk": 128,
         "dv": 128, "per_token": True},
        # ragged prompts in f32, keys shared by two value heads, one constant decay per head
        {"name": "linear_ragged_5x_f32", "op": "linear", "dtype": F32, "B": 5, "lo": 1, "hi": 1500, "pick": 8, "nh": 16, "nkh": 8, "dk": 64,
         "dv": 128, "per_token": False},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    top_bytes = max(work(c)["bytes"] for c in listed())
    top_flops = max(work(c)["flops"] for c in listed())
    while True:
        case = _draw(rng)
        w = work(case)
        if w["bytes"] <= top_bytes and w["flops"] <= top_flops * (1.0 if case["dtype"] == BF16 else 0.25):
            return case


def _draw(rng):
    op = rng.choice(["norm_rope", "kv4_store", "kv4_attn", "kv4_attn", "linear", "linear_step"])
    case = {"op": op, "dtype": rng.choice([F32, BF16, BF16]), "pick": rng.randrange(1 << 20)}
    if op == "norm_rope":
        nh, nkv, hd, rot = rng.choice([(96, 96, 192, 64), (64, 8, 128, 128), (32, 8, 64, 32), (16, 1, 256, 64), (40, 8, 128, 64), (64, 1, 512, 64)])
        case.update(T=_log_int(rng, 1, 8192), nh=nh, nkv=nkv, hd=hd, rot=rot, halves=rng.random() < 0.5)
        return case
    if op == "linear" or op == "linear_step":
        nh, nkh, dk, dv = rng.choice([(32, 32, 128, 128), (16, 16, 64, 64), (16, 8, 64, 128), (32, 8, 128, 64), (24, 24, 128, 128)])
        case.update(B=_log_int(rng, 1, 64 if op == "linear_step" else 8), nh=nh, nkh=nkh, dk=dk, dv=dv, per_token=rng.random() < 0.7)
        if op == "linear":
            hi = _log_int(rng, 2, 8192)
            case.update(lo=rng.choice([1, hi]), hi=hi)
        return case
    nh, nkv, dk, rope, dv = rng.choice([(96, 96, 128, 64, 128), (64, 8, 128, 0, 128), (32, 8, 64, 0, 64), (16, 2, 256, 0, 256), (40, 8, 128, 0, 128),
                                        (48, 3, 128, 64, 128)])
    case.update(nkv=nkv, dk=dk, rope=rope, dv=dv)
    if op == "kv4_store":
        hi = _log_int(rng, 1, 2048)
        case.update(B=_log_int(rng, 1, 16), lo=rng.choice([1, hi]), hi=hi)
        return case
    rows = rng.choice([1, 1, 1, rng.randrange(2, 9), _log_int(rng, 9, 512)])
    hi = _log_int(rng, rows, 16384)
    case.update(B=_log_int(rng, 1, 32), lo=rng.choice([rows, hi]), hi=hi, rows=rows, nh=nh)
    return case


def _lens(case):
    """The sequences' lengths: fixed by the case, spread over their logarithm, the longest always among them."""
    rng = random.Random(case["pick"])
    out = [_log_int(rng, case["lo"], case["hi"]) for _ in range(case["B"])]
    out[rng.randrange(case["B"])] = case["hi"]
    return out


def work(case):
    e, op = _bytes_of(case), case["op"]
    if op == "norm_rope":
        n = case["T"] * (case["nh"] + case["nkv"]) * case["hd"]
        return {"bytes": 2 * n * e + case["T"] * (case["rot"] * 4 + 4) + 2 * case["hd"] * 4, "flops": 7 * n}
    if op == "linear_step":
        n, st = case["B"] * case["nh"], case["dk"] * case["dv"]
        rows = case["B"] * (2 * case["nkh"] * case["dk"] + 2 * case["nh"] * case["dv"])
        return {"bytes": 8 * n * st + rows * e, "flops": 5 * n * st}
    if op == "linear":
        lens = _lens(case)
        T, st = sum(lens), case["dk"] * case["dv"]
        rows = T * (2 * case["nkh"] * case["dk"] + 2 * case["nh"] * case["dv"])
        return {"bytes": rows * e + 8 * case["B"] * case["nh"] * st + (4 * T * case["nh"] if case["per_token"] else 0), "flops": 4 * T * case["nh"] * st}
    lens = _lens(case)
    held = case["nkv"] * (case["dk"] + case["dv"]) * 17 // 32 + 2 * case["rope"]  # bytes of one position
    if op == "kv4_store":
        row = case["nkv"] * (case["dk"] + case["rope"] + case["dv"])
        return {"bytes": sum(lens) * (row * e + 2 * held) + 4 * row * case["B"] * case["hi"], "flops": 6 * sum(lens) * row}
    rows, nh = case["rows"], case["nh"]
    pairs = sum(rows * n - rows * (rows - 1) // 2 for n in lens)
    width = case["dk"] + case["rope"] + case["dv"]
    return {"bytes": sum(lens) * held + case["B"] * rows * nh * width * e, "flops": 2 * pairs * nh * width}


# ------------------------------------------------------------------------------------------------------------ the inputs

def _normal(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen, device="cuda").to(dtype)


def _cu(lens):
    return torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device="cuda")


def _codes(x):
    """MXFP4 of x [..., n]: bytes [..., n/2] (low nibble = even value) and e8m0 bytes [..., n/32].  The exponent is the
    smallest e with 6 * 2^e >= the block's largest magnitude, the level the nearest one, upwards at a midpoint."""
    b = x.float().reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    m, ex = torch.frexp(b.abs().amax(-1))
    e = torch.where(m == 0, torch.full_like(ex, -127), torch.where(m <= 0.75, ex - 3, ex - 2)).clamp(-127, 125)
    a = torch.ldexp(b.abs(), -e.unsqueeze(-1))
    lev = torch.zeros_like(a, dtype=torch.uint8)
    for mid in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0):
        lev += (a >= mid).to(torch.uint8)
    lev = (lev | ((b < 0).to(torch.uint8) << 3)).reshape(*x.shape[:-1], x.shape[-1] // 2, 2)
    return lev[..., 0] | (lev[..., 1] << 4), (e + 127).to(torch.uint8)


def _values(packed, scales):
    """f32 values of MXFP4 bytes."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=packed.device)
    nib = torch.stack((packed & 15, packed >> 4), -1).reshape(*packed.shape[:-1], packed.shape[-1] * 2)
    v = table[nib.int()].reshape(*scales.shape, 32)
    return torch.ldexp(v, scales.int().unsqueeze(-1) - 127).reshape(nib.shape)


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt, op = _dt(case), case["op"]
    st = {"case": case}
    if op == "norm_rope":
        T, nh, nkv, hd, rot = (case[k] for k in ("T", "nh", "nkv", "hd", "rot"))
        # the projections' output: q and k of a token side by side in one row, as a fused projection leaves them
        qk = _normal(gen, T, nh + nkv, hd, dtype=dt)
        st.update(q=qk[:, :nh], k=qk[:, nh:], wq=1 + 0.1 * _normal(gen, hd), wk=1 + 0.1 * _normal(gen, hd), eps=1e-6)
        n_pos = 32768
        freq = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
        ang = torch.arange(n_pos, dtype=torch.float64, device="cuda")[:, None] * freq
        st.update(cos=ang.cos().float(), sin=ang.sin().float())
        first = int(torch.randint(0, n_pos - T + 1, (1,), generator=gen, device="cuda"))
        st["pos"] = torch.arange(first, first + T, dtype=torch.int32, device="cuda")
        return st
    if op in ("linear", "linear_step"):
        lens = _lens(case) if op == "linear" else [1] * case["B"]
        T, B, nh, nkh, dk, dv = sum(lens), case["B"], case["nh"], case["nkh"], case["dk"], case["dv"]
        st.update(lens=lens, cu=_cu(lens) if op == "linear" and B > 1 else None, q=_normal(gen, T, nkh, dk, dtype=dt), k=_normal(gen, T, nkh, dk, dtype=dt),
                  v=_normal(gen, T, nh, dv, dtype=dt), state=_normal(gen, B, nh, dk, dv), scale=dk ** -0.5)
        # log decays: slow and fast heads; per token the softplus form of a gate
        if case["per_token"]:
            speed = torch.exp(torch.linspace(-5.0, 0.0, nh, device="cuda"))
            st["g"] = -speed * torch.nn.functional.softplus(_normal(gen, T, nh))
        else:
            st["g"] = -torch.exp(torch.linspace(-6.0, -1.0, nh, device="cuda")) * (1 + 0.1 * torch.rand(nh, generator=gen, device="cuda"))
        st["out"], st["state_out"] = torch.empty_like(st["v"]), torch.empty_like(st["state"])
        return st
    lens = _lens(case)
    B, nkv, dk, rope, dv, cap = case["B"], case["nkv"], case["dk"], case["rope"], case["dv"], case["hi"]
    st["lens"] = lens
    if op == "kv4_store":
        T = sum(lens)
        st.update(k=_normal(gen, T, nkv, dk + rope, dtype=dt), v=_normal(gen, T, nkv, dv, dtype=dt), cu=_cu(lens))
        return st
    # the cache of sequences that were pushed earlier: MXFP4 rows of N(0, 1) keys and values, bfloat16 rope rows
    kq = torch.empty((B, nkv, cap, dk // 2), dtype=torch.uint8, device="cuda")
    ks = torch.empty((B, nkv, cap, dk // 32), dtype=torch.uint8, device="cuda")
    vq = torch.empty((B, nkv, cap, dv // 2), dtype=torch.uint8, device="cuda")
    vs = torch.empty((B, nkv, cap, dv // 32), dtype=torch.uint8, device="cuda")
    for b in range(B):
        kq[b], ks[b] = _codes(_normal(gen, nkv, cap, dk))
        vq[b], vs[b] = _codes(_normal(gen, nkv, cap, dv))
    kr = _normal(gen, B, cap, rope, dtype=torch.bfloat16) if rope else None
    st.update(q=_normal(gen, B * case["rows"], case["nh"], dk + rope, dtype=dt), scale=(dk + rope) ** -0.5, kq=kq, ks=ks, kr=kr, vq=vq, vs=vs)
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    if own and case["op"].startswith("kv4"):
        from microkimi_amd import mixer
        if case["op"] == "kv4_store":
            st["cache"] = mixer.KvCache4(case["B"], case["nkv"], case["dk"], case["dv"], case["hi"], rope=case["rope"])
        else:
            st["cache"] = mixer.KvCache4.from_parts(st["kq"], st["ks"], st["kr"], st["vq"], st["vs"],
                                                    torch.tensor(st["lens"], dtype=torch.int32, device="cuda"))
    return st


# ------------------------------------------------------------------------------------------------------ one pass of each

def run(state):
    op = state["case"]["op"]
    return (_own if own else _plain)[op](state)


def _norm_rope_own(s):
    from microkimi_amd import mixer
    return mixer.qk_norm_rope(s["q"], s["k"], s["cos"], s["sin"], s["pos"], wq=s["wq"], wk=s["wk"], eps=s["eps"], halves=s["case"]["halves"])


def _kv4_store_own(s):
    s["cache"].assign(s["k"], s["v"], cu=s["cu"])
    return s["cache"].to_f32(s["case"]["hi"])


def _kv4_attn_own(s):
    return s["cache"].attn(s["q"], s["scale"])


def _linear_own(s):
    from microkimi_amd import mixer
    return mixer.linear_attn(s["q"], s["k"], s["v"], s["g"], s["state"], s["scale"], cu=s["cu"], out=s["out"], state_out=s["state_out"])


def _linear_step_own(s):
    from microkimi_amd import mixer
    return mixer.linear_attn_step(s["q"], s["k"], s["v"], s["g"], s["state"], s["scale"], out=s["out"], state_out=s["state_out"])


def _norm_rope_plain(s):
    rot, hd = s["case"]["rot"], s["case"]["hd"]
    c, sn = s["cos"][s["pos"].long()][:, None], s["sin"][s["pos"].long()][:, None]
    outs = []
    for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
        y = x.float()
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + s["eps"]) * w
        head, r = y[..., :hd - rot], y[..., hd - rot:]
        if s["case"]["halves"]:
            a, b = r[..., :rot // 2], r[..., rot // 2:]
            r = torch.cat((a * c - b * sn, a * sn + b * c), -1)
        else:
            a, b = r[..., 0::2], r[..., 1::2]
            r = torch.stack((a * c - b * sn, a * sn + b * c), -1).flatten(-2)
        outs.append(torch.cat((head, r), -1).to(x.dtype))
    return tuple(outs)


def _kv4_store_plain(s):
    case = s["case"]
    nkv, dk, rope, n = case["nkv"], case["dk"], case["rope"], case["hi"]
    k = torch.zeros((case["B"], n, nkv, dk + rope), device="cuda")
    v = torch.zeros((case["B"], n, nkv, case["dv"]), device="cuda")
    kv = _values(*_codes(s["k"][..., :dk]))
    vv = _values(*_codes(s["v"]))
    t0 = 0
    for b, m in enumerate(s["lens"]):
        k[b, :m, :, :dk], v[b, :m] = kv[t0:t0 + m], vv[t0:t0 + m]
        if rope:  # one row for all heads, the first head's, held in bfloat16
            k[b, :m, :, dk:] = s["k"][t0:t0 + m, :1, dk:].bfloat16().float()
        t0 += m
    return k, v


def _kv4_attn_plain(s):
    case = s["case"]
    nh, nkv, dk, rope, rows = case["nh"], case["nkv"], case["dk"], case["rope"], case["rows"]
    outs = []
    for b, n in enumerate(s["lens"]):
        q = s["q"][b * rows:(b + 1) * rows].float().transpose(0, 1).reshape(nkv, nh // nkv * rows, dk + rope)
        k = _values(s["kq"][b, :, :n], s["ks"][b, :, :n])
        if rope:
            k = torch.cat((k, s["kr"][b, None, :n].float().expand(nkv, n, rope)), -1)
        sc = torch.matmul(q, k.transpose(1, 2).contiguous()) * s["scale"]
        if rows > 1:
            limit = torch.arange(n - rows, n, device="cuda").repeat(nh // nkv)
            sc.masked_fill_(torch.arange(n, device="cuda")[None] > limit[:, None], -math.inf)
        p = torch.exp(sc - sc.amax(-1, keepdim=True))
        o = torch.matmul(p, _values(s["vq"][b, :, :n], s["vs"][b, :, :n])) / p.sum(-1, keepdim=True)
        outs.append(o.reshape(nh, rows, case["dv"]).transpose(0, 1))
    return torch.cat(outs).to(s["q"].dtype)


def _linear_plain(s):
    """Blocks of 256 tokens: inside a block as a masked product, across blocks through the state."""
    nh, C = s["case"]["nh"], 256
    rep = nh // s["case"]["nkh"]
    out, states, t0 = torch.empty_like(s["v"]), s["state"].clone(), 0
    for b, n in enumerate(s["lens"]):
        S = states[b]
        for c0 in range(t0, t0 + n, C):
            c1 = min(c0 + C, t0 + n)
            q, k, v = (x[c0:c1].float().transpose(0, 1) for x in (s["q"], s["k"], s["v"]))
            q, k = q.repeat_interleave(rep, 0), k.repeat_interleave(rep, 0)
            g = s["g"][c0:c1].T if s["case"]["per_token"] else s["g"][:, None].expand(nh, c1 - c0)
            cum = g.double().cumsum(-1)
            dec = torch.exp((cum[:, :, None] - cum[:, None, :]).float()).tril()
            o = torch.matmul(torch.matmul(q, k.transpose(1, 2).contiguous()) * dec, v) + torch.exp(cum.float())[..., None] * torch.matmul(q, S)
            out[c0:c1] = (o * s["scale"]).transpose(0, 1).to(out.dtype)
            kd = k * torch.exp((cum[:, -1:] - cum).float())[..., None]
            S = torch.exp(cum[:, -1].float())[:, None, None] * S + torch.matmul(kd.transpose(1, 2).contiguous(), v)
        states[b] = S
        t0 += n
    return out, states


def _linear_step_plain(s):
    rep = s["case"]["nh"] // s["case"]["nkh"]
    q, k = s["q"].float().repeat_interleave(rep, 1), s["k"].float().repeat_interleave(rep, 1)
    g = s["g"] if s["case"]["per_token"] else s["g"][None]
    S = torch.exp(g)[..., None, None] * s["state"] + k[..., None] * s["v"].float()[..., None, :]
    return ((q[..., None] * S).sum(-2) * s["scale"]).to(s["v"].dtype), S


_own = {"norm_rope": _norm_rope_own, "kv4_store": _kv4_store_own, "kv4_attn": _kv4_attn_own, "linear": _linear_own, "linear_step": _linear_step_own}
_plain = {"norm_rope": _norm_rope_plain, "kv4_store": _kv4_store_plain, "kv4_attn": _kv4_attn_plain, "linear": _linear_plain,
          "linear_step": _linear_step_plain}


# ------------------------------------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    s = _inputs(case, seed)
    return {"norm_rope": _norm_rope_exact, "kv4_store": _kv4_store_exact, "kv4_attn": _kv4_attn_exact, "linear": _linear_exact,
            "linear_step": _linear_exact}[case["op"]](case, s)


def _norm_rope_exact(case, s):
    rot, outs = case["rot"], []
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["pos"].long()][:, None]
    for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
        y = x.double().clone()
        y *= w.double() * (y.square().sum(-1, keepdim=True) / case["hd"] + s["eps"]).rsqrt()
        r = y[..., -rot:]
        if case["halves"]:
            z = torch.complex(r[..., :rot // 2].contiguous(), r[..., rot // 2:].contiguous()) * turn
            y[..., -rot:] = torch.cat((z.real, z.imag), -1)
        else:
            z = torch.view_as_complex(r.reshape(*r.shape[:-1], rot // 2, 2).contiguous()) * turn
            y[..., -rot:] = torch.view_as_real(z).reshape(r.shape)
        outs.append(y)
    return tuple(outs)


def _mxfp4_exact(x):
    """The nearest of the 16 values of each block's grid, by distance."""
    b = x.double().reshape(*x.shape[:-1], -1, 32)
    top = b.abs().amax(-1, keepdim=True)
    e = torch.full_like(top, -127.0)
    for k in range(-126, 126):
        e = torch.where(6.0 * 2.0 ** (k - 1) < top, torch.full_like(top, float(k)), e)
    step = torch.pow(2.0, e)
    a = b.abs() / step
    # below 2 the levels are 0.5 apart, from 2 to 4 they are 1 apart, above 2
    q = torch.where(a < 2, torch.floor(a * 2 + 0.5) / 2, torch.where(a < 4, torch.floor(a + 0.5), torch.floor(a / 2 + 0.5) * 2)).clamp(max=6)
    return (torch.sign(b) * q * step).reshape(x.shape)


def _kv4_store_exact(case, s):
    dk, rope, n = case["dk"], case["rope"], case["hi"]
    parts = [], []
    for kb, vb in zip(s["k"].split(s["lens"]), s["v"].split(s["lens"])):
        k = [_mxfp4_exact(kb[..., :dk])]
        if rope:
            k.append(kb[:, 0:1, dk:].bfloat16().double().expand(-1, case["nkv"], -1))
        pad = (0, 0, 0, 0, 0, n - kb.shape[0])
        parts[0].append(torch.nn.functional.pad(torch.cat(k, -1), pad))
        parts[1].append(torch.nn.functional.pad(_mxfp4_exact(vb), pad))
    return torch.stack(parts[0]), torch.stack(parts[1])


def _levels64(packed, scales):
    lo, hi = packed & 15, packed >> 4
    nib = torch.stack((lo, hi), -1).flatten(-2).long()
    mag = nib & 7
    val = torch.where(mag < 2, 0.5 * mag.double(), (1 + 0.5 * (mag & 1).double()) * torch.pow(2.0, (mag >> 1).double() - 1))
    val = torch.where(nib > 7, -val, val)
    return val * torch.pow(2.0, scales.double() - 127).repeat_interleave(32, -1)


def _kv4_attn_exact(case, s):
    nh, nkv, rope, rows = case["nh"], case["nkv"], case["rope"], case["rows"]
    group, out = nh // nkv, torch.empty((case["B"] * rows, nh, case["dv"]), dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lens"]):
        hidden = torch.arange(n, device="cuda")[None] > torch.arange(n - rows, n, device="cuda")[:, None]
        for j in range(nkv):
            k, v = _levels64(s["kq"][b, j, :n], s["ks"][b, j, :n]), _levels64(s["vq"][b, j, :n], s["vs"][b, j, :n])
            if rope:
                k = torch.cat((k, s["kr"][b, :n].double()), -1)
            for h in range(j * group, (j + 1) * group):
                sc = s["scale"] * (s["q"][b * rows:(b + 1) * rows, h].double() @ k.T)
                out[b * rows:(b + 1) * rows, h] = torch.softmax(sc.masked_fill(hidden, -math.inf), -1) @ v
    return out


def _linear_exact(case, s):
    """Token by token, all sequences side by side; a sequence that has ended keeps its state."""
    B, nh, rep = case["B"], case["nh"], case["nh"] // case["nkh"]
    S, out, lens = s["state"].double().clone(), torch.empty(s["v"].shape, dtype=torch.float64, device="cuda"), s["lens"]
    starts = [sum(lens[:b]) for b in range(B)]
    order = sorted(range(B), key=lambda b: -lens[b])
    S = S[order].contiguous()
    for t in range(max(lens)):
        live = sum(1 for b in order if lens[b] > t)
        if live == 1:
            row = slice(starts[order[0]] + t, starts[order[0]] + t + 1)
        else:
            row = torch.tensor([starts[b] + t for b in order[:live]], device="cuda")
        q, k, v = s["q"][row].double(), s["k"][row].double(), s["v"][row].double()
        if rep > 1:
            q, k = q.repeat_interleave(rep, 1), k.repeat_interleave(rep, 1)
        g = s["g"][row].double() if case["per_token"] else s["g"].double()[None].expand(live, nh)
        S[:live] = S[:live] * torch.exp(g)[..., None, None] + k[..., None] * v[..., None, :]
        out[row] = s["scale"] * (q[..., None, :] @ S[:live])[..., 0, :]
    back = torch.empty_like(S)
    back[order] = S
    return out, back
