"""The token mixers of a layer beside the MLA cache of model.py: head norm + rotation of queries and keys, attention over a KV
cache held in 4 bits (several sequences, grouped-query heads), and linear attention with a decay for each head.

Rows are f32 or bfloat16 tensors on the current device, [tokens, heads, width]; a token's heads must lie one behind the other, the
tokens may be further apart (slices of one projection's rows are taken as they are, other layouts are copied).  A batch of
sequences: rows one sequence behind the other, cu [B + 1] int32 on the device = where each one's rows begin (None: equally many
rows each).  Outputs that the caller gives must not overlap the inputs, except where a call says that it works in place.  Every call
only enqueues work on the current stream and takes what it needs from torch's allocator, so calls may be captured into graphs and run
on several streams."""
import ctypes as C

import torch

from . import _lib
from ._lib import BF16, F32, Kv4Cache, check, lib

_TYPES = {torch.float32: F32, torch.bfloat16: BF16}
_F32 = torch.float32
_bound = False

# torch's internal forms of the calls after them (0.08 instead of 1.15 us, 0.11 instead of 0.22), where it has them
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda dev: torch.cuda.current_stream(dev).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _start(ref):
    """The current stream of the device that the call's tensors are on, which has to be the current one."""
    global _bound
    if not _bound:
        _lib.require_device()
        _bound = True
    dev = ref.get_device()
    if dev != _current_device():
        raise ValueError(f"tensors are on cuda:{dev}, the current device is cuda:{_current_device()}")
    return _raw_stream(dev)


def _code(t):
    if not t.is_cuda:
        raise ValueError("tensors must be on the GPU")
    dt = _TYPES.get(t.dtype)
    if dt is None:
        raise ValueError("rows must be float32 or bfloat16")
    return dt


def _rows(t, name, width=None):
    """(tensor, values from one token to the next) of rows [T, heads, width]."""
    if t.dim() != 3 or (width is not None and t.shape[2] != width):
        raise ValueError(f"{name} must be [tokens, heads, {width or 'width'}], not {tuple(t.shape)}")
    T, h, w = t.shape
    if t.is_contiguous() and not t.data_ptr() & 15:
        return t, h * w
    s0, s1, s2 = t.stride()
    if (s2 != 1 and w > 1) or (s1 != w and h > 1) or (T > 1 and (s0 % 8 or s0 < h * w)) or t.data_ptr() & 15:
        t = t.contiguous()
        if t.data_ptr() & 15:
            t = t.clone()
        return t, h * w
    return t, s0 if T > 1 else h * w


def _same(ref, t, name, dtype=None):
    if t.dtype != (dtype or ref.dtype):
        raise ValueError(f"{name} must be {dtype or ref.dtype}, not {t.dtype}")
    if t.get_device() != ref.get_device():
        raise ValueError(f"{name} is on {t.device}, not on {ref.device}")


def _f32(ref, t, name, shape=None):
    if t.dtype is not _F32 or t.get_device() != ref.get_device():
        _same(ref, t, name, _F32)
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} must be {tuple(shape)}, not {tuple(t.shape)}")
    if t.is_contiguous() and not t.data_ptr() & 15:
        return t
    t = t.contiguous()
    return t if not t.data_ptr() & 15 else t.clone()


def _result(out, ref, shape, name, dtype=None):
    """The caller's output tensor after its checks, or a new one."""
    if out is None:
        if dtype is None:
            return torch.empty_like(ref, memory_format=torch.contiguous_format) if shape == ref.shape else ref.new_empty(shape)
        return ref.new_empty(shape, dtype=dtype)
    _same(ref, out, name, dtype)
    if out.shape != shape or not out.is_contiguous() or out.data_ptr() & 15:
        raise ValueError(f"{name} must be a contiguous, 16-byte aligned {tuple(shape)} tensor")
    return out


def _apart(out, name, *inputs):
    """Refuses an output of the caller's that begins where an input begins which other workgroups may still read."""
    at = out.data_ptr()
    for t in inputs:
        if t is not None and t.data_ptr() == at and at:
            raise ValueError(f"{name} must not overlap the call's inputs")


def _workspace(ref, n):
    """(n bytes of device memory for a call, their address), or none."""
    if n == 0:
        return None, None
    ws = torch.empty(n, dtype=torch.uint8, device=ref.device)
    return ws, ws.data_ptr()


def _cu_ptr(ref, cu, B, T):
    if cu is None:
        if T % B:
            raise ValueError(f"{T} rows do not divide among {B} sequences: give cu")
        return None
    _same(ref, cu, "cu", torch.int32)
    if cu.dim() != 1 or cu.shape[0] != B + 1 or not cu.is_contiguous():
        raise ValueError(f"cu must be {B + 1} contiguous values")
    return cu.data_ptr()


def _ptr(t):
    return None if t is None else t.data_ptr()


def rope_table(n_pos, rot, base=10000.0, device="cuda"):
    """(cos, sin) [n_pos, rot / 2] f32 of the angles pos * base^(-2 i / rot), formed in 64 bits (far positions keep their angle)."""
    freq = float(base) ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot)
    ang = torch.arange(n_pos, dtype=torch.float64, device=device)[:, None] * freq
    return ang.cos().float(), ang.sin().float()


def qk_norm_rope(q, k, cos=None, sin=None, pos=None, wq=None, wk=None, eps=1e-6, norm=True, rot_at=None, halves=False, q_out=None, k_out=None):
    """RMS norm of every query head (q [T, nh, hd]) and key head (k [T, nkv, hd], or None) with the rotation of the token's
    position in the same pass (mk_dev_qk_norm_rope).  wq, wk [hd] f32 or None (ones); norm=False leaves the norm out.  cos, sin
    [n_pos, rot / 2] f32 (rope_table), pos [T] int32; rot_at: first rotated value of a head (default: the last rot values);
    pairs (2 i, 2 i + 1), or (i, i + rot / 2) with halves=True.  A negative position marks a padding row, which is not
    written.  Returns (q_out, k_out); q_out=q, k_out=k work in place (contiguous rows)."""
    ref = q if q is not None else k
    if ref is None:
        raise ValueError("q or k must be given")
    dt, hd, T = _code(ref), ref.shape[-1], ref.shape[0]
    rot = n_pos = 0
    if cos is not None:
        if sin is None or pos is None:
            raise ValueError("a rotation needs cos, sin and pos")
        if cos.dim() != 2 or sin.shape != cos.shape:
            raise ValueError("cos and sin must be [n_pos, rot / 2]")
        n_pos, rot = cos.shape
        rot *= 2
        cos, sin = _f32(ref, cos, "cos"), _f32(ref, sin, "sin")
    if pos is not None:
        _same(ref, pos, "pos", torch.int32)
        if pos.dim() != 1 or pos.shape[0] != T or not pos.is_contiguous():
            raise ValueError(f"pos must be {T} contiguous values")
    if q_out is not None:
        _apart(q_out, "q_out", k)
    if k_out is not None:
        _apart(k_out, "k_out", q, q_out)
    qr, qp, qs, nh, wq, wqp, qo, qop = _heads(ref, q, wq, q_out, T, hd, "q")
    kr, kp, ks, nkv, wk, wkp, ko, kop = _heads(ref, k, wk, k_out, T, hd, "k")
    check(lib.mk_dev_qk_norm_rope(dt, qp, qs, nh, kp, ks, nkv, T, hd, 1 if norm else 0, wqp, wkp, eps, _ptr(cos), _ptr(sin), n_pos, _ptr(pos), rot,
                                  hd - rot if rot_at is None else rot_at, 1 if halves else 0, qop, nh * hd, kop, nkv * hd, _start(ref)))
    return qo, ko


def _heads(ref, x, w, out, T, hd, name):
    """(rows, their address, token stride, heads, weights, their address, output rows, their address) of one side of qk_norm_rope."""
    if x is None:
        return None, None, 0, 0, None, None, None, None
    if x is not ref:
        _same(ref, x, name)
        if x.shape[0] != T:
            raise ValueError("q and k must have the same tokens")
    xr, stride = _rows(x, name, hd)
    if w is not None:
        w = _f32(ref, w, "w" + name, (hd,))
    out = _result(out, x, x.shape, name + "_out")
    return xr, xr.data_ptr(), stride, x.shape[1], w, None if w is None else w.data_ptr(), out, out.data_ptr()


class KvCache4:
    """A KV cache held in 4 bits for B sequences of up to `capacity` positions (mk_kv4_cache): per kv head K rows of dk and V rows
    of dv values as MXFP4, and a K tail of `rope` values that the heads share (rows as model.MlaHeadsCache takes them: the tail
    last, taken from head 0) in bfloat16.  lens [B] int32 on the device counts the positions held and moves with every push, also
    inside a captured graph."""

    def __init__(self, B, nkv, dk, dv, capacity, rope=0, device="cuda"):
        if dk % 32 or dv % 32 or not (32 <= dk <= 512 and 32 <= dv <= 512):
            raise ValueError("K and V widths must be multiples of 32 up to 512")
        if rope % 8 or not 0 <= rope <= 64:
            raise ValueError("the shared K tail must be a multiple of 8 up to 64")
        if B < 1 or nkv < 1 or capacity < 1:
            raise ValueError("B, nkv and capacity must be positive")
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
        if kq.dim() != 4 or vq.dim() != 4:
            raise ValueError("kq and vq must be [B, nkv, capacity, width / 2]")
        B, nkv, cap, dk, dv = *kq.shape[:3], 2 * kq.shape[3], 2 * vq.shape[3]
        rope = kr.shape[-1] if kr is not None else 0
        for t, shape, dt, name in ((kq, (B, nkv, cap, dk // 2), torch.uint8, "kq"), (ks, (B, nkv, cap, dk // 32), torch.uint8, "ks"),
                                   (vq, (B, nkv, cap, dv // 2), torch.uint8, "vq"), (vs, (B, nkv, cap, dv // 32), torch.uint8, "vs"),
                                   (kr, (B, cap, rope), torch.bfloat16, "kr"), (lens, (B,), torch.int32, "lens")):
            if t is None and name == "kr":
                continue
            _same(kq, t, name, dt)
            if t.shape != shape or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous {shape} tensor")
        self.B, self.nkv, self.dk, self.dv, self.rope, self.cap = B, nkv, dk, dv, rope, cap
        self.kq, self.ks, self.kr, self.vq, self.vs, self.lens = kq, ks, kr, vq, vs, lens
        self.table = Kv4Cache(B, nkv, dk, rope, dv, cap, kq.data_ptr(), ks.data_ptr(), vq.data_ptr(), vs.data_ptr(), kr.data_ptr() if rope else None,
                              lens.data_ptr())
        self._ref = C.byref(self.table)
        self._f32 = lens.new_empty(0, dtype=torch.float32)   # (what new f32 tensors are made like)

    def positions(self):
        """Positions held by each sequence (waits for the device)."""
        return self.lens.tolist()

    def _store(self, k_rows, v_rows, cu, fresh):
        dt = _code(k_rows)
        _same(self.lens, k_rows, "k_rows", k_rows.dtype)
        _same(k_rows, v_rows, "v_rows")
        T = k_rows.shape[0]
        if k_rows.dim() != 3 or k_rows.shape[1] != self.nkv:
            raise ValueError(f"k_rows must be [rows, {self.nkv}, {self.dk + self.rope}]")
        if v_rows.dim() != 3 or v_rows.shape[:2] != (T, self.nkv):
            raise ValueError(f"v_rows must be [{T}, {self.nkv}, {self.dv}]")
        k_rows, ks = _rows(k_rows, "k_rows", self.dk + self.rope)
        v_rows, vs = _rows(v_rows, "v_rows", self.dv)
        cup = _cu_ptr(k_rows, cu, self.B, T)
        check(lib.mk_dev_kv4_append(self._ref, dt, k_rows.data_ptr(), ks, v_rows.data_ptr(), vs, T, cup, fresh, _start(k_rows)))

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
        n = self.cap if n is None else n
        if not 0 <= n <= self.cap:
            raise ValueError("more positions than the cache holds")
        k = self._f32.new_empty((self.B, n, self.nkv, self.dk + self.rope))
        v = self._f32.new_empty((self.B, n, self.nkv, self.dv))
        check(lib.mk_dev_kv4_to_f32(self._ref, n, k.data_ptr(), v.data_ptr(), _start(k)))
        return k, v

    def attn(self, q, scale, cu=None, max_len=None, out=None):
        """Softmax attention of the rows pushed last: q [T, nh, dk + rope], the m rows of a sequence are its last m positions, each
        attends what lies before it and itself (one row: a decode step; a prompt: causal).  nh a multiple of nkv.  Returns
        [T, nh, dv].  max_len: an upper bound of the sequences' lengths, if the caller keeps one (steers the split of the work
        only, which goes by the capacity without it: worth giving where that is many times what is held)."""
        dt = _code(q)
        _same(self.lens, q, "q", q.dtype)
        q, stride = _rows(q, "q", self.dk + self.rope)
        T, nh = q.shape[:2]
        if nh % self.nkv or nh == 0:
            raise ValueError(f"the query heads must be a multiple of {self.nkv}")
        cup = _cu_ptr(q, cu, self.B, T)
        out = _result(out, q, (T, nh, self.dv), "out")
        ws, wp = _workspace(q, lib.mk_kv4_attn_workspace_bytes(self._ref, T, nh))
        check(lib.mk_dev_kv4_attn(self._ref, dt, q.data_ptr(), stride, T, cup, nh, scale, max_len or 0, wp, out.data_ptr(), _start(q)))
        return out


def _linear_args(q, k, v, g, state, B, out, state_out):
    dt = _code(q)
    _same(q, k, "k")
    _same(q, v, "v")
    if q.dim() != 3 or k.shape != q.shape:
        raise ValueError("k must have the shape of q, [tokens, key heads, dk]")
    if v.dim() != 3 or v.shape[0] != q.shape[0]:
        raise ValueError("v must be [tokens, value heads, dv]")
    T, nkh, dk = q.shape
    nh, dv = v.shape[1:]
    if nkh == 0 or nh == 0 or nh % nkh:
        raise ValueError("the value heads must be a multiple of the key heads")
    _same(q, g, "g", torch.float32)
    if g.dim() == 1:
        if g.shape[0] != nh:
            raise ValueError(f"g must be [{nh}] or [{T}, {nh}]")
        g, gs = g.contiguous(), 0
    else:
        if g.shape != (T, nh):
            raise ValueError(f"g must be [{nh}] or [{T}, {nh}]")
        if (nh > 1 and g.stride(1) != 1) or (T > 1 and g.stride(0) < nh):
            g = g.contiguous()
        gs = g.stride(0) if T > 1 else nh
    shape = (B, nh, dk, dv)
    if state_out is not None:
        _apart(state_out, "state_out", q, k, v)
    if out is not None:
        _apart(out, "out", q, k, state, state_out)
    if state is not None:
        state = _f32(q, state, "state", shape)
    state_out = _result(state_out, q, shape, "state_out", torch.float32)
    out = _result(out, v, v.shape, "out")
    (q, qs), (k, ks), (v, vs) = _rows(q, "q"), _rows(k, "k"), _rows(v, "v")
    return dt, q, qs, k, ks, v, vs, g, gs, T, nh, nkh, dk, dv, state, state_out, out


def linear_attn(q, k, v, g, state=None, scale=1.0, cu=None, B=None, out=None, state_out=None):
    """Linear attention with a decay for each head over whole prompts (mk_dev_linear_attn): per value head
    S_t = exp(g_t) S_{t-1} + k_t v_t^T, o_t = scale * S_t^T q_t.  q, k [T, nkh, dk], v [T, nh, dv], g [T, nh] (log decays f32) or [nh]
    (constant), state [B, nh, dk, dv] f32 or None (zeros).  B: the number of sequences (default: cu's, or state's, or 1).
    Returns (out [T, nh, dv], state_out); state_out=state updates in place."""
    if B is None:
        B = cu.shape[0] - 1 if cu is not None else state.shape[0] if state is not None else 1
    if B < 1:
        raise ValueError("there must be a sequence")
    dt, q, qs, k, ks, v, vs, g, gs, T, nh, nkh, dk, dv, state, state_out, out = _linear_args(q, k, v, g, state, B, out, state_out)
    cup = _cu_ptr(q, cu, B, T)
    ws, wp = _workspace(q, lib.mk_linear_attn_workspace_bytes(T, B, nh, dk, dv))
    check(lib.mk_dev_linear_attn(dt, q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, g.data_ptr(), gs, T, cup, B, nh, nkh, dk, dv, scale,
                                 None if state is None else state.data_ptr(), state_out.data_ptr(), wp, out.data_ptr(), _start(q)))
    return out, state_out


def linear_attn_step(q, k, v, g, state=None, scale=1.0, out=None, state_out=None):
    """linear_attn for one token of each of B sequences (mk_dev_linear_attn_step): q, k [B, nkh, dk], v [B, nh, dv], g [B, nh] or
    [nh], state [B, nh, dk, dv].  Returns (out [B, nh, dv], state_out)."""
    dt, q, qs, k, ks, v, vs, g, gs, B, nh, nkh, dk, dv, state, state_out, out = _linear_args(q, k, v, g, state, q.shape[0], out, state_out)
    if B == 0:
        return out, state_out
    check(lib.mk_dev_linear_attn_step(dt, q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, g.data_ptr(), gs, B, nh, nkh, dk, dv, scale,
                                      None if state is None else state.data_ptr(), state_out.data_ptr(), out.data_ptr(), _start(q)))
    return out, state_out
