"""What the token-mixer calls refuse, without a device: the C ABI on made-up pointers (nothing is launched), the Python layer on
CPU tensors."""
import ctypes as C

import pytest
import torch

from microkimi_amd import mixer
from microkimi_amd._lib import Kv4Cache, lib

P = 4096  # an aligned address that is never read


def refused(status, *words):
    assert status == -1
    text = lib.mk_last_error().decode()
    assert all(w in text for w in words), text


def norm_rope(dtype=0, q=P, qs=256, nh=2, k=P, ks=256, nkv=2, T=3, hd=128, norm=1, wq=None, wk=None, cos=P, sin=P, n_pos=8, pos=P, rot=64, rot_at=64, qo=P, qos=256,
              ko=P, kos=256):
    return lib.mk_dev_qk_norm_rope(dtype, q, qs, nh, k, ks, nkv, T, hd, norm, wq, wk, 1e-6, cos, sin, n_pos, pos, rot, rot_at, 0, qo, qos, ko, kos, None)


@pytest.mark.parametrize("bad,word", [(dict(dtype=2), "dtype"), (dict(q=None), "null"), (dict(ko=None), "null"), (dict(hd=12), "multiple of 8"),
                                      (dict(hd=520), "512"), (dict(rot=24), "16"), (dict(rot_at=72), "inside"), (dict(rot_at=4), "of 8"),
                                      (dict(rot_at=2 ** 63), "inside"), (dict(pos=None), "positions"), (dict(qs=255), "multiples of 8"),
                                      (dict(ks=248), "shorter"), (dict(kos=128), "shorter"), (dict(q=P + 8), "aligned"), (dict(wk=P + 4), "aligned"),
                                      (dict(cos=P + 8), "aligned"), (dict(T=2 ** 31), "range")])
def test_norm_rope_refusals(bad, word):
    refused(norm_rope(**bad), word)


def cache(B=2, nkv=2, dk=128, rope=64, dv=128, cap=64, kq=P, ks=P, vq=P, vs=P, kr=P, lens=P):
    return C.byref(Kv4Cache(B, nkv, dk, rope, dv, cap, kq, ks, vq, vs, kr, lens))


CACHES = [(dict(kq=None), "null"), (dict(kr=None), "null"), (dict(lens=None), "null"), (dict(dk=48), "32"), (dict(dv=0), "32"), (dict(dv=544), "512"),
          (dict(rope=12), "tail"), (dict(rope=72), "tail"), (dict(cap=0), "capacity"), (dict(cap=2 ** 23), "capacity"), (dict(B=0), "count"),
          (dict(nkv=70000), "count"), (dict(vq=P + 8), "aligned")]


@pytest.mark.parametrize("bad,word", CACHES)
def test_cache_refusals(bad, word):
    c = cache(**bad)
    refused(lib.mk_dev_kv4_append(c, 0, P, 4096, P, 4096, 2, None, 0, None), word)
    refused(lib.mk_dev_kv4_to_f32(c, 4, P, P, None), word)
    refused(lib.mk_dev_kv4_attn(c, 0, P, 4096, 2, None, 2, 1.0, 0, P, P, None), word)


def test_append_snapshot_and_attention_refusals():
    c = cache()
    refused(lib.mk_dev_kv4_append(None, 0, P, 384, P, 256, 2, None, 0, None), "null")
    refused(lib.mk_dev_kv4_append(c, 3, P, 384, P, 256, 2, None, 0, None), "dtype")
    refused(lib.mk_dev_kv4_append(c, 0, P, 384, P, 256, 3, None, 0, None), "same number")
    refused(lib.mk_dev_kv4_append(c, 0, P, 376, P, 256, 2, None, 0, None), "shorter")
    refused(lib.mk_dev_kv4_append(c, 0, P, 384, P, 250, 2, None, 0, None), "multiples of 8")
    refused(lib.mk_dev_kv4_append(c, 0, P + 4, 384, P, 256, 2, None, 0, None), "aligned")
    refused(lib.mk_dev_kv4_append(c, 0, None, 384, P, 256, 2, None, 0, None), "null")
    refused(lib.mk_dev_kv4_append(c, 0, P, 384, P, 256, 2 ** 22, P, 0, None), "rows")
    refused(lib.mk_dev_kv4_to_f32(c, 65, P, P, None), "more positions")
    refused(lib.mk_dev_kv4_to_f32(c, 64, P, P + 4, None), "aligned")
    refused(lib.mk_dev_kv4_attn(c, 0, P, 384, 2, None, 3, 1.0, 0, P, P, None), "multiple of the kv heads")
    refused(lib.mk_dev_kv4_attn(c, 0, P, 384, 3, None, 2, 1.0, 0, P, P, None), "same number")
    refused(lib.mk_dev_kv4_attn(c, 0, P, 384, 2, None, 4, 1.0, 0, P, P, None), "shorter")
    refused(lib.mk_dev_kv4_attn(c, 0, P, 384, 2, None, 2, 1.0, 0, P + 16, P, None), "workspace")
    refused(lib.mk_dev_kv4_attn(c, 0, P, 384, 2, None, 2, 1.0, 0, P, None, None), "null")
    long = cache(cap=4096)
    assert lib.mk_kv4_attn_workspace_bytes(long, 2, 2) > 0
    refused(lib.mk_dev_kv4_attn(long, 0, P, 384, 2, None, 2, 1.0, 0, None, P, None), "null")
    assert lib.mk_dev_kv4_attn(c, 0, None, 384, 0, None, 2, 1.0, 0, None, None, None) == 0   # no rows: nothing to do
    assert lib.mk_kv4_attn_workspace_bytes(c, 1, 96) == 0      # one piece: nothing to keep


def linear(dtype=0, q=P, qs=256, k=P, ks=256, v=P, vs=256, g=P, gs=2, T=4, cu=None, B=2, nh=2, nkh=2, dk=128, dv=128, state=P, state_out=P, ws=P, out=P):
    return lib.mk_dev_linear_attn(dtype, q, qs, k, ks, v, vs, g, gs, T, cu, B, nh, nkh, dk, dv, 1.0, state, state_out, ws, out, None)


@pytest.mark.parametrize("bad,word", [(dict(dtype=9), "dtype"), (dict(B=0), "count"), (dict(T=5), "same number"), (dict(nkh=0), "key heads"), (dict(nh=3), "key heads"),
                                      (dict(dk=4), "multiples of 8"), (dict(dv=264), "256"), (dict(v=None), "null"), (dict(state_out=None), "null"),
                                      (dict(g=None), "null"), (dict(qs=250), "multiples of 8"), (dict(vs=248), "shorter"), (dict(gs=1), "shorter"),
                                      (dict(k=P + 8), "aligned"), (dict(state=P + 4), "aligned"), (dict(ws=None, T=2048), "workspace"), (dict(ws=P + 16), "workspace")])
def test_linear_refusals(bad, word):
    refused(linear(**bad), word)
    if not {"T", "ws"} & set(bad):
        a = dict(dtype=0, q=P, qs=256, k=P, ks=256, v=P, vs=256, g=P, gs=2, B=2, nh=2, nkh=2, dk=128, dv=128, state=P, state_out=P, out=P)
        a.update(bad)
        refused(lib.mk_dev_linear_attn_step(a["dtype"], a["q"], a["qs"], a["k"], a["ks"], a["v"], a["vs"], a["g"], a["gs"], a["B"], a["nh"], a["nkh"], a["dk"],
                                            a["dv"], 1.0, a["state"], a["state_out"], a["out"], None), word)


def test_off_switch_comes_first():
    lib.mk_set_enabled(0)
    try:
        assert norm_rope(dtype=7) == -2 and linear(dtype=7) == -2
        assert lib.mk_dev_kv4_append(None, 0, P, 384, P, 256, 2, None, 0, None) == -2
    finally:
        lib.mk_set_enabled(1)


def test_python_layer_refuses_cpu_tensors_and_wrong_shapes():
    x = torch.zeros(2, 4, 128)
    with pytest.raises(ValueError, match="GPU"):
        mixer.qk_norm_rope(x, None)
    with pytest.raises(ValueError, match="q or k"):
        mixer.qk_norm_rope(None, None)
    with pytest.raises(ValueError, match="GPU"):
        mixer.linear_attn(x, x, x, torch.zeros(2, 4))
    with pytest.raises(ValueError, match="multiples of 32"):
        mixer.KvCache4(1, 1, 40, 64, 8, device="cpu")
    with pytest.raises(ValueError, match="tail"):
        mixer.KvCache4(1, 1, 64, 64, 8, rope=4, device="cpu")
    c = mixer.KvCache4(1, 1, 64, 64, 8, device="cpu")
    with pytest.raises(ValueError, match="GPU"):
        c.push(torch.zeros(1, 1, 64), torch.zeros(1, 1, 64))
    with pytest.raises(ValueError, match="GPU"):
        c.attn(torch.zeros(1, 2, 64), 1.0)
    with pytest.raises(ValueError, match="capacity|positions"):
        c.to_f32(9)
    with pytest.raises(ValueError, match="lens"):
        mixer.KvCache4.from_parts(c.kq, c.ks, None, c.vq, c.vs, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="ks"):
        mixer.KvCache4.from_parts(c.kq, c.ks[..., :1], None, c.vq, c.vs, c.lens)


def test_tables_hold_far_positions():
    cos, sin = mixer.rope_table(1 << 17, 64, device="cpu")
    import math
    for p in (0, 1, 70001, (1 << 17) - 1):
        for i in (0, 1, 31):
            a = p * 10000.0 ** (-2 * i / 64)
            assert abs(float(cos[p, i]) - math.cos(a)) <= 2 ** -24 + 1e-9 and abs(float(sin[p, i]) - math.sin(a)) <= 2 ** -24 + 1e-9


def test_the_cache_struct_is_the_same_in_the_header_the_binding_and_the_shim():
    import pathlib
    import re
    root = pathlib.Path(__file__).resolve().parents[1]
    body = re.search(r"typedef struct \{([^}]*)\} mk_kv4_cache;", (root / "include/mk_hip.h").read_text()).group(1)
    header = []
    for kind, names in re.findall(r"(\w+) ([^;]+);", body):
        header += [(n.strip(" *"), "*" in n, kind) for n in names.split(",")]
    body = re.search(r"struct MkKv4Cache \{([^}]*)\}", (root / "rust/hip.rs").read_text()).group(1)
    rust = [(n, t.startswith("*mut"), t.split()[-1]) for n, t in re.findall(r"(\w+): ([^,\n]+)", body)]
    kinds = {"size_t": "usize", "uint8_t": "u8", "uint16_t": "u16", "int32_t": "i32"}
    assert rust == [(n, p, kinds[k]) for n, p, k in header]
    assert [(n, t is C.c_size_t) for n, t in Kv4Cache._fields_] == [(n, not p) for n, p, _ in header]


def test_the_package_imports_where_torch_lacks_its_internal_names():
    """The host entry points need neither a stream nor a device."""
    import os
    import pathlib
    import subprocess
    import sys
    code = ("import torch\n"
            "for n in ('_cuda_getCurrentRawStream', '_cuda_getDevice'):\n"
            "    if hasattr(torch._C, n): delattr(torch._C, n)\n"
            "import microkimi_amd\n"
            "print(microkimi_amd._lib.lib.mk_enabled_now(), callable(microkimi_amd.mixer.qk_norm_rope))\n")
    root = str(pathlib.Path(__file__).resolve().parents[1])
    run = subprocess.run([sys.executable, "-c", code], cwd=root, env=dict(os.environ, PYTHONPATH=root), stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert run.returncode == 0, run.stdout
    assert run.stdout.split()[-2:] == ["1", "True"]
