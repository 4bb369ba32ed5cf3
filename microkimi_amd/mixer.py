"""The token mixers of a layer beside the MLA cache of model.py: head norm + rotation of queries and keys, attention over a KV
cache held in 4 bits (several sequences, grouped-query heads), and linear attention with a decay for each head.

Rows are f32 or bfloat16 tensors on the current device, [tokens, heads, width]; a token's heads must lie one behind the other, the
tokens may be further apart (slices of one projection's rows are taken as they are, other layouts are copied).  A batch of
sequences: rows one sequence behind the other, cu [B + 1] int32 on the device = where each one's rows begin (None: equally many
rows each).  Every call only enqueues work on the current stream and takes what it needs from torch's allocator, so calls may
be captured into graphs and run on several streams."""
import ctypes as C

from . import _lib
from ._lib import BF16, F32, Kv4Cache, check, lib


def _need(cond, msg):
    if not cond:
        raise ValueError(msg)


def _stream(device):
    import torch
    _need(device.index == torch.cuda.current_device(), f"tensors are on {device}, the current device is cuda:{torch.cuda.current_device()}")
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _code(t):
    import torch
    _need(t.is_cuda, "tensors must be on the GPU")
    if t.dtype == torch.float32:
        return F32
    _need(t.dtype == torch.bfloat16, "rows must be float32 or bfloat16")
    return BF16


def _rows(t, name, width=None):
    """(tensor, values from one token to the next) of rows [T, heads, width]."""
    _need(t.dim() == 3 and (width is None or t.shape[2] == width), f"{name} must be [tokens, heads, {width or 'width'}]")
    T, h, w = t.shape
    s = t.stride()
    if (s[2] != 1 and w > 1) or (s[1] != w and h > 1) or s[0] % 8 or (T > 1 and s[0] < h * w) or t.data_ptr() & 15:
        t = t.contiguous()
        if t.data_ptr() & 15:
            t = t.clone()
        return t, h * w
    return t, s[0] if T > 1 else h * w


def _same(ref, t, name, dtype=None):
    _need(t.device == ref.device, f"{name} is on {t.device}, not on {ref.device}")
    _need(t.dtype == (dtype or ref.dtype), f"{name} must be {dtype or ref.dtype}")


def _f32(ref, t, name, shape=None):
    import torch
    _same(ref, t, name, torch.float32)
    _need(shape is None or tuple(t.shape) == shape, f"{name} must be {shape}")
    t = t.contiguous()
    return t if not t.data_ptr() & 15 else t.clone()


def _result(out, ref, shape, name):
    """The caller's output tensor after its checks, or a new one."""
    import torch
    if out is None:
        return torch.empty(shape, dtype=ref.dtype, device=ref.device)
    _same(ref, out, name)
    _need(tuple(out.shape) == tuple(shape) and out.is_contiguous() and not out.data_ptr() & 15, f"{name} must be a contiguous, 16-byte aligned {tuple(shape)} tensor")
    return out


def _cu_ptr(ref, cu, B, T):
    import torch
    if cu is None:
        _need(T % B == 0, f"{T} rows do not divide among {B} sequences: give cu")
        return None
    _same(ref, cu, "cu", torch.int32)
    _need(cu.dim() == 1 and cu.shape[0] == B + 1 and cu.is_contiguous(), f"cu must be {B + 1} contiguous values")
    return cu.data_ptr()


def rope_table(n_pos, rot, base=10000.0, device="cuda"):
    """(cos, sin) [n_pos, rot / 2] f32 of the angles pos * base^(-2 i / rot), formed in 64 bits (far positions keep their angle)."""
    import torch
    freq = float(base) ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot)
    ang = torch.arange(n_pos, dtype=torch.float64, device=device)[:, None] * freq
    return ang.cos().float(), ang.sin().float()


def qk_norm_rope(q, k, cos=None, sin=None, pos=None, wq=None, wk=None, eps=1e-6, norm=True, rot_at=None, halves=False, q_out=None, k_out=None):
    """RMS norm of every query head (q [T, nh, hd]) and key head (k [T, nkv, hd], or None) with the rotation of the token's
    position in the same pass (mk_dev_qk_norm_rope).  wq, wk [hd] f32 or None (ones); norm=False leaves the norm out.  cos, sin
    [n_pos, rot / 2] f32 (rope_table), pos [T] int32; rot_at: first rotated value of a head (default: the last rot values);
    pairs (2 i, 2 i + 1), or (i, i + rot / 2) with halves=True.  A negative position marks a padding row, which is not
    written.  Returns (q_out, k_out); q_out=q, k_out=k work in place (contiguous rows)."""
    import torch
    ref = q if q is not None else k
    _need(ref is not None, "q or k must be given")
    dt, hd, T = _code(ref), ref.shape[-1], ref.shape[0]
    rot = 2 * cos.shape[1] if cos is not None else 0
    if rot:
        _need(sin is not None and pos is not None, "a rotation needs cos, sin and pos")
        _need(cos.dim() == 2 and sin.shape == cos.shape, "cos and sin must be [n_pos, rot / 2]")
        cos, sin = _f32(ref, cos, "cos"), _f32(ref, sin, "sin")
    if pos is not None:
        _same(ref, pos, "pos", torch.int32)
        _need(pos.dim() == 1 and pos.shape[0] == T and pos.is_contiguous(), "pos must be [T]")
    args, outs = [], []
    for x, w, o, name in ((q, wq, q_out, "q"), (k, wk, k_out, "k")):
        if x is None:
            args.append((None, 0, 0, None, None, 0))
            outs.append(None)
            continue
        _same(ref, x, name)
        _need(x.shape[0] == T, "q and k must have the same tokens")
        h = x.shape[1] if x.dim() == 3 else 0
        o = _result(o, x, x.shape, f"{name}_out")
        xr, stride = _rows(x, name, hd)
        w = _f32(ref, w, f"w{name}", (hd,)) if w is not None else None
        args.append((xr, stride, h, w, o, h * hd))
        outs.append(o)
    (qr, qs, nh, wq, qo, qos), (kr, ks, nkv, wk, ko, kos) = args
    _lib.require_device()
    p = lambda t: None if t is None else t.data_ptr()
    check(lib.mk_dev_qk_norm_rope(dt, p(qr), qs, nh, p(kr), ks, nkv, T, hd, int(bool(norm)), p(wq), p(wk), eps, p(cos), p(sin), cos.shape[0] if rot else 0,
                                  p(pos), rot, hd - rot if rot_at is None else rot_at, int(bool(halves)), p(qo), qos, p(ko), kos, _stream(ref.device)))
    return outs[0], outs[1]


class KvCache4:
    """A KV cache held in 4 bits for B sequences of up to `capacity` positions (mk_kv4_cache): per kv head K rows of dk and V rows
    of dv values as MXFP4, and a K tail of `rope` values that the heads share (rows as model.MlaHeadsCache takes them: the tail
    last, taken from head 0) in bfloat16.  lens [B] int32 on the device counts the positions held and moves with every push, also
    inside a captured graph."""

    def __init__(self, B, nkv, dk, dv, capacity, rope=0, device="cuda"):
        import torch
        _need(dk % 32 == 0 and dv % 32 == 0 and 32 <= dk <= 512 and 32 <= dv <= 512, "K and V widths must be multiples of 32 up to 512")
        _need(rope % 8 == 0 and 0 <= rope <= 64, "the shared K tail must be a multiple of 8 up to 64")
        _need(B >= 1 and nkv >= 1 and capacity >= 1, "B, nkv and capacity must be positive")
        z = lambda *shape: torch.zeros(shape, dtype=torch.uint8, device=device)
        kr = torch.zeros((B, capacity, rope), dtype=torch.bfloat16, device=device) if rope else None
        self._bind(z(B, nkv, capacity, dk // 2), z(B, nkv, capacity, dk // 32), kr, z(B, nkv, capacity, dv // 2), z(B, nkv, capacity, dv // 32),
                   torch.zeros(B, dtype=torch.int32, device=device))

    @staticmethod
    def from_parts(kq, ks, kr, vq, vs, lens):
        """A cache over existing arrays (layout: mk_kv4_cache; kr None: no shared tail), as a snapshot or another program left them."""
        c = KvCache4.__new__(KvCache4)
        c._bind(kq, ks, kr, vq, vs, lens)
        return c

    def _bind(self, kq, ks, kr, vq, vs, lens):
        import torch
        _need(kq.dim() == 4 and vq.dim() == 4, "kq and vq must be [B, nkv, capacity, width / 2]")
        B, nkv, cap, dk, dv = *kq.shape[:3], 2 * kq.shape[3], 2 * vq.shape[3]
        rope = kr.shape[-1] if kr is not None else 0
        for t, shape, dt, name in ((kq, (B, nkv, cap, dk // 2), torch.uint8, "kq"), (ks, (B, nkv, cap, dk // 32), torch.uint8, "ks"),
                                   (vq, (B, nkv, cap, dv // 2), torch.uint8, "vq"), (vs, (B, nkv, cap, dv // 32), torch.uint8, "vs"),
                                   (kr, (B, cap, rope), torch.bfloat16, "kr"), (lens, (B,), torch.int32, "lens")):
            if t is None and name == "kr":
                continue
            _same(kq, t, name, dt)
            _need(tuple(t.shape) == shape and t.is_contiguous(), f"{name} must be a contiguous {shape} tensor")
        self.B, self.nkv, self.dk, self.dv, self.rope, self.cap = B, nkv, dk, dv, rope, cap
        self.kq, self.ks, self.kr, self.vq, self.vs, self.lens = kq, ks, kr, vq, vs, lens
        self.table = Kv4Cache(B, nkv, dk, rope, dv, cap, kq.data_ptr(), ks.data_ptr(), vq.data_ptr(), vs.data_ptr(), kr.data_ptr() if rope else None,
                              lens.data_ptr())
        self._ref = C.byref(self.table)

    def positions(self):
        """Positions held by each sequence (waits for the device)."""
        return self.lens.tolist()

    def _store(self, k_rows, v_rows, cu, fresh):
        dt = _code(k_rows)
        _same(self.lens, k_rows, "k_rows", k_rows.dtype)
        _same(k_rows, v_rows, "v_rows")
        T = k_rows.shape[0]
        _need(k_rows.dim() == 3 and k_rows.shape[1] == self.nkv, f"k_rows must be [rows, {self.nkv}, {self.dk + self.rope}]")
        _need(v_rows.dim() == 3 and tuple(v_rows.shape[:2]) == (T, self.nkv), f"v_rows must be [{T}, {self.nkv}, {self.dv}]")
        k_rows, ks = _rows(k_rows, "k_rows", self.dk + self.rope)
        v_rows, vs = _rows(v_rows, "v_rows", self.dv)
        cup = _cu_ptr(k_rows, cu, self.B, T)
        _lib.require_device()
        check(lib.mk_dev_kv4_append(self._ref, dt, k_rows.data_ptr(), ks, v_rows.data_ptr(), vs, T, cup, fresh, _stream(k_rows.device)))

    def push(self, k_rows, v_rows, cu=None):
        """Rows k_rows [T, nkv, dk + rope], v_rows [T, nkv, dv] behind what each sequence holds (MlaCache::push for a batch).  A row
        beyond the capacity is not stored; a query that would have to attend one gives NaN."""
        self._store(k_rows, v_rows, cu, 0)

    def assign(self, k_rows, v_rows, cu=None):
        """The sequences emptied, then filled (MlaCache::assign_f32 for a batch)."""
        self._store(k_rows, v_rows, cu, 1)

    def to_f32(self, n=None):
        """The values of the first n positions (default: all the capacity): k [B, n, nkv, dk + rope], v [B, n, nkv, dv] f32, zeros
        where a sequence holds none."""
        import torch
        n = self.cap if n is None else n
        _need(0 <= n <= self.cap, "more positions than the cache holds")
        k = torch.empty((self.B, n, self.nkv, self.dk + self.rope), dtype=torch.float32, device=self.lens.device)
        v = torch.empty((self.B, n, self.nkv, self.dv), dtype=torch.float32, device=self.lens.device)
        _lib.require_device()
        check(lib.mk_dev_kv4_to_f32(self._ref, n, k.data_ptr(), v.data_ptr(), _stream(k.device)))
        return k, v

    def attn(self, q, scale, cu=None, max_len=None, out=None):
        """Softmax attention of the rows pushed last: q [T, nh, dk + rope], the m rows of a sequence are its last m positions, each
        attends what lies before it and itself (one row: a decode step; a prompt: causal).  nh a multiple of nkv.  Returns
        [T, nh, dv].  max_len: an upper bound of the sequences' lengths, if the caller keeps one (steers the split of the work
        only)."""
        import torch
        dt = _code(q)
        _same(self.lens, q, "q", q.dtype)
        q, stride = _rows(q, "q", self.dk + self.rope)
        T, nh = q.shape[:2]
        _need(nh % self.nkv == 0 and nh > 0, f"the query heads must be a multiple of {self.nkv}")
        cup = _cu_ptr(q, cu, self.B, T)
        out = _result(out, q, (T, nh, self.dv), "out")
        _lib.require_device()
        ws = torch.empty(lib.mk_kv4_attn_workspace_bytes(self._ref, T, nh), dtype=torch.uint8, device=q.device)
        check(lib.mk_dev_kv4_attn(self._ref, dt, q.data_ptr(), stride, T, cup, nh, scale, max_len or 0, ws.data_ptr(), out.data_ptr(), _stream(q.device)))
        return out


def _linear_args(q, k, v, g, state, B, out, state_out):
    import torch
    dt = _code(q)
    _same(q, k, "k")
    _same(q, v, "v")
    _need(q.dim() == 3 and k.shape == q.shape, "k must have the shape of q, [tokens, key heads, dk]")
    _need(v.dim() == 3 and v.shape[0] == q.shape[0], "v must be [tokens, value heads, dv]")
    T, nkh, dk = q.shape
    nh, dv = v.shape[1:]
    _need(nkh > 0 and nh % nkh == 0, "the value heads must be a multiple of the key heads")
    _same(q, g, "g", torch.float32)
    if g.dim() == 1:
        _need(g.shape[0] == nh, f"g must be [{nh}] or [{T}, {nh}]")
        g, gs = g.contiguous(), 0
    else:
        _need(tuple(g.shape) == (T, nh), f"g must be [{nh}] or [{T}, {nh}]")
        if (nh > 1 and g.stride(1) != 1) or (T > 1 and g.stride(0) < nh):
            g = g.contiguous()
        gs = g.stride(0) if T > 1 else nh
    shape = (B, nh, dk, dv)
    if state is not None:
        state = _f32(q, state, "state", shape)
    if state_out is None:
        state_out = torch.empty(shape, dtype=torch.float32, device=q.device)
    else:
        _same(q, state_out, "state_out", torch.float32)
        _need(tuple(state_out.shape) == shape and state_out.is_contiguous() and not state_out.data_ptr() & 15, f"state_out must be a contiguous {shape} tensor")
    out = _result(out, v, v.shape, "out")
    (q, qs), (k, ks), (v, vs) = _rows(q, "q"), _rows(k, "k"), _rows(v, "v")
    return dt, q, qs, k, ks, v, vs, g, gs, T, nh, nkh, dk, dv, state, state_out, out


def linear_attn(q, k, v, g, state=None, scale=1.0, cu=None, B=None, out=None, state_out=None):
    """Linear attention with a decay for each head over whole prompts (mk_dev_linear_attn): per value head
    S_t = exp(g_t) S_{t-1} + k_t v_t^T, o_t = scale * S_t^T q_t.  q, k [T, nkh, dk], v [T, nh, dv], g [T, nh] (log decays f32) or [nh]
    (constant), state [B, nh, dk, dv] f32 or None (zeros).  B: the number of sequences (default: cu's, or state's, or 1).
    Returns (out [T, nh, dv], state_out); state_out=state updates in place."""
    import torch
    if B is None:
        B = cu.shape[0] - 1 if cu is not None else state.shape[0] if state is not None else 1
    dt, q, qs, k, ks, v, vs, g, gs, T, nh, nkh, dk, dv, state, state_out, out = _linear_args(q, k, v, g, state, B, out, state_out)
    cup = _cu_ptr(q, cu, B, T)
    _lib.require_device()
    ws = torch.empty(lib.mk_linear_attn_workspace_bytes(T, B, nh, dk, dv), dtype=torch.uint8, device=q.device)
    check(lib.mk_dev_linear_attn(dt, q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, g.data_ptr(), gs, T, cup, B, nh, nkh, dk, dv, scale,
                                 None if state is None else state.data_ptr(), state_out.data_ptr(), ws.data_ptr(), out.data_ptr(), _stream(q.device)))
    return out, state_out


def linear_attn_step(q, k, v, g, state=None, scale=1.0, out=None, state_out=None):
    """linear_attn for one token of each of B sequences (mk_dev_linear_attn_step): q, k [B, nkh, dk], v [B, nh, dv], g [B, nh] or
    [nh], state [B, nh, dk, dv].  Returns (out [B, nh, dv], state_out)."""
    dt, q, qs, k, ks, v, vs, g, gs, B, nh, nkh, dk, dv, state, state_out, out = _linear_args(q, k, v, g, state, q.shape[0], out, state_out)
    _lib.require_device()
    check(lib.mk_dev_linear_attn_step(dt, q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, g.data_ptr(), gs, B, nh, nkh, dk, dv, scale,
                                      None if state is None else state.data_ptr(), state_out.data_ptr(), out.data_ptr(), _stream(q.device)))
    return out, state_out
