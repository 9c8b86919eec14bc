"""vireo-b200: vireo's MoE FFN hot path, B200-native (sm_100a).

The product is the C-ABI shared library ``libvireo_b200.so`` built from
``csrc/`` (headers in ``include/``).  This package loads it with ctypes and
mirrors the reference interface for Python callers:

* ``gguf_matmul`` / ``gguf_dequant_row`` / ``gguf_f16_to_f32`` — the three
  functions of the reference's gguf_compute.h (vireo src/gguf_compute.h:8-10);
* ``MoeLayer`` — the MoE FFN block (reference moe_ffn, src/gguf_run.c:185-214)
  behind ``gguf_moe_*``;
* ``kv_plan`` and ``PagedKV`` — many requests over one paged key-value pool
  (the reference's KV store seam, src/kvstore.h:48-71) behind ``gguf_kv_*``.

There is no fallback: if the library is missing or no CUDA device is
present, calls raise.
"""
from __future__ import annotations

import ctypes as C
import os
import struct
import subprocess

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libvireo_b200.so")

VIREO_OK = 0
STATUS = {0: "ok", -1: "invalid argument", -2: "CUDA runtime error", -3: "unsupported tensor type or shape",
          -4: "device wait timed out", -5: "out of memory", -6: "I/O error", -7: "no CUDA device"}


class VireoError(RuntimeError):
    def __init__(self, status: int, what: str = ""):
        super().__init__(f"{what}: {STATUS.get(status, status)} ({status})")
        self.status = status


def build(jobs: int = 8) -> str:
    """Compile libvireo_b200.so for sm_100a (nvcc cross-compiles without a GPU)."""
    subprocess.run(["make", "-s", "-C", HERE, f"-j{jobs}"], check=True)
    return LIB_PATH


class GgufTensor(C.Structure):
    """gguf_tensor (reference src/gguf.h:36-45), ABI-identical."""
    _fields_ = [("name_ptr", C.c_char_p), ("name_len", C.c_uint64), ("n_dims", C.c_uint32),
                ("dims", C.c_uint64 * 4), ("ggml_type", C.c_uint32), ("offset", C.c_uint64),
                ("data", C.c_void_p), ("n_elems", C.c_uint64), ("nbytes", C.c_uint64)]


class GgufMoeDesc(C.Structure):
    _fields_ = [("dim", C.c_int), ("ffn_exp", C.c_int), ("n_experts", C.c_int), ("n_used", C.c_int),
                ("topk_renorm", C.c_int), ("router_type", C.c_uint32), ("gate_type", C.c_uint32),
                ("up_type", C.c_uint32), ("down_type", C.c_uint32), ("router", C.c_void_p),
                ("gate_exps", C.c_void_p), ("up_exps", C.c_void_p), ("down_exps", C.c_void_p),
                ("gate_nbytes", C.c_uint64), ("up_nbytes", C.c_uint64), ("down_nbytes", C.c_uint64)]


class GgufMoeShexpDesc(C.Structure):
    _fields_ = [("dim", C.c_int), ("ffn", C.c_int), ("gate_type", C.c_uint32), ("up_type", C.c_uint32),
                ("down_type", C.c_uint32), ("gate", C.c_void_p), ("up", C.c_void_p), ("down", C.c_void_p),
                ("gate_inp", C.c_void_p)]


class ExpertStats(C.Structure):
    _fields_ = [(n, C.c_uint64) for n in ("requests", "hits", "misses", "bytes_read", "resident_bytes",
                                          "capacity_bytes", "experts_resident")]


class ExpertSlices(C.Structure):
    _fields_ = [("gate_off", C.c_uint64), ("up_off", C.c_uint64), ("down_off", C.c_uint64),
                ("gate_bytes", C.c_uint32), ("up_bytes", C.c_uint32), ("down_bytes", C.c_uint32)]


class ExpertView(C.Structure):
    _fields_ = [("gate", C.c_void_p), ("up", C.c_void_p), ("down", C.c_void_p), ("slot", C.c_void_p)]


class ExpertStatsExt(C.Structure):
    _fields_ = [(n, C.c_uint64) for n in ("h2d_bytes", "copies", "evictions", "over_budget_loads")]


_lib = None


def lib():
    """The loaded C-ABI library (raises if it was never built)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise FileNotFoundError(f"{LIB_PATH} is missing: run vireo_b200.build() (no CPU fallback exists)")
        L = C.CDLL(LIB_PATH)
        L.gguf_f16_to_f32.argtypes = [C.c_uint16]
        L.gguf_f16_to_f32.restype = C.c_float
        L.gguf_dequant_row.argtypes = [C.c_uint32, C.c_void_p, C.c_void_p, C.c_int]
        L.gguf_dequant_row.restype = None
        L.gguf_matmul.argtypes = [C.c_void_p, C.c_void_p, C.POINTER(GgufTensor), C.c_int, C.c_int]
        L.gguf_matmul.restype = None
        L.vireo_last_error.restype = C.c_int
        L.vireo_status_string.argtypes = [C.c_int]
        L.vireo_status_string.restype = C.c_char_p
        L.vireo_device_init.argtypes = [C.c_int]
        L.gguf_matmul_dev.argtypes = [C.c_void_p, C.c_void_p, C.POINTER(GgufTensor), C.c_int, C.c_int, C.c_void_p]
        L.gguf_dequant_row_dev.argtypes = [C.c_uint32, C.c_void_p, C.c_void_p, C.c_int, C.c_void_p]
        L.gguf_weights_register.argtypes = [C.c_void_p, C.c_uint64]
        L.gguf_weights_unregister.argtypes = [C.c_void_p]
        L.vireo_sync.argtypes = [C.c_void_p]
        L.gguf_moe_create.argtypes = [C.POINTER(GgufMoeDesc), C.POINTER(C.c_void_p)]
        L.gguf_moe_ffn.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, C.c_void_p, C.c_void_p]
        L.gguf_moe_ffn_host.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, C.c_void_p]
        L.gguf_moe_sync.argtypes = [C.c_void_p, C.c_void_p]
        L.gguf_moe_set_expert_ptrs.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p]
        L.gguf_moe_destroy.argtypes = [C.c_void_p]
        L.gguf_moe_shexp_create.argtypes = [C.POINTER(GgufMoeShexpDesc), C.POINTER(C.c_void_p)]
        L.gguf_moe_shexp_ffn.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_void_p]
        L.gguf_moe_shexp_sync.argtypes = [C.c_void_p, C.c_void_p]
        L.gguf_moe_shexp_destroy.argtypes = [C.c_void_p]
        L.gguf_moe_ffn_noalloc.argtypes = [C.POINTER(GgufMoeDesc), C.c_void_p, C.c_void_p, C.c_int, C.c_void_p,
                                           C.c_void_p, C.c_void_p]
        L.gguf_moe_destroy.restype = None
        L.gguf_moe_ffn_routed.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, C.c_void_p,
                                          C.c_void_p, C.c_void_p]
        L.gguf_moe_ffn_store.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, C.c_void_p, C.c_void_p,
                                         C.c_void_p, C.c_void_p]
        L.gguf_moe_prefill.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, C.c_void_p,
                                       C.c_void_p, C.c_void_p]
        # expert parallelism (include/gguf_moe.h)
        L.gguf_moe_ep_unique_id.argtypes = [C.c_void_p]
        L.gguf_moe_ep_place.argtypes = [C.c_void_p, C.c_int, C.c_int, C.c_void_p]
        L.gguf_moe_ep_rows.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_void_p, C.c_void_p]
        L.gguf_moe_ep_create.argtypes = [C.POINTER(GgufMoeDesc), C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_void_p,
                                         C.POINTER(C.c_void_p)]
        L.gguf_moe_prefill_ep.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, C.c_void_p,
                                          C.c_void_p, C.c_void_p]
        L.gguf_moe_ep_sync.argtypes = [C.c_void_p, C.c_void_p]
        L.gguf_moe_ep_layer.argtypes = [C.c_void_p]
        L.gguf_moe_ep_layer.restype = C.c_void_p
        L.gguf_moe_ep_destroy.argtypes = [C.c_void_p]
        L.gguf_moe_ep_destroy.restype = None
        # ExpertStore (include/expert_store.h)
        L.expert_store_create.argtypes = [C.c_int, C.c_uint64, C.c_int, C.c_int]
        L.expert_store_create.restype = C.c_void_p
        L.expert_store_create_host.argtypes = [C.c_void_p, C.c_uint64, C.c_uint64, C.c_int, C.c_int]
        L.expert_store_create_host.restype = C.c_void_p
        L.expert_store_register.argtypes = [C.c_void_p, C.c_int, C.c_int, C.POINTER(ExpertSlices)]
        L.expert_store_register.restype = None
        L.expert_store_lookup.argtypes = [C.c_void_p, C.c_int, C.c_int, C.POINTER(ExpertView)]
        L.expert_store_lookup_async.argtypes = [C.c_void_p, C.c_int, C.c_int, C.POINTER(ExpertView), C.c_void_p]
        L.expert_store_release.argtypes = [C.c_void_p, C.POINTER(ExpertView)]
        L.expert_store_release.restype = None
        L.expert_store_release_after.argtypes = [C.c_void_p, C.POINTER(ExpertView), C.c_void_p]
        L.expert_store_stats.argtypes = [C.c_void_p, C.POINTER(ExpertStats)]
        L.expert_store_stats.restype = None
        L.expert_store_stats_ext.argtypes = [C.c_void_p, C.POINTER(ExpertStatsExt)]
        L.expert_store_stats_ext.restype = None
        L.expert_store_destroy.argtypes = [C.c_void_p]
        L.expert_store_destroy.restype = None
        _lib = L
    return _lib


def check(status: int, what: str) -> None:
    if status != VIREO_OK:
        raise VireoError(status, what)


def _ptr(a) -> int:
    """Address of a numpy array or torch tensor."""
    if isinstance(a, np.ndarray):
        return a.ctypes.data
    return a.data_ptr()


# ---------------------------------------------------------------------------
# gguf_compute.h mirror
# ---------------------------------------------------------------------------

def gguf_f16_to_f32(h: int) -> float:
    return lib().gguf_f16_to_f32(h)


def gguf_dequant_row(ggml_type: int, src, n: int, out=None):
    """Reference gguf_dequant_row; src/out numpy (host) or torch CUDA tensors."""
    if out is None:
        out = np.zeros(n, dtype=np.float32)
    lib().gguf_dequant_row(ggml_type, _ptr(src), _ptr(out), n)
    check(lib().vireo_last_error(), "gguf_dequant_row")
    return out


def make_tensor(ggml_type: int, data) -> GgufTensor:
    t = GgufTensor()
    t.ggml_type = ggml_type
    t.data = _ptr(data)
    return t


def gguf_matmul(ggml_type: int, w, x, n: int, d: int, y=None):
    """Reference gguf_matmul: y[d] = W[d x n] . x[n] (host or device buffers)."""
    if y is None:
        y = np.zeros(d, dtype=np.float32)
    t = make_tensor(ggml_type, w)
    lib().gguf_matmul(_ptr(y), _ptr(x), C.byref(t), n, d)
    check(lib().vireo_last_error(), "gguf_matmul")
    return y


def gguf_matmul_dev(ggml_type: int, w, x, n: int, d: int, y, stream=None) -> None:
    t = make_tensor(ggml_type, w)
    check(lib().gguf_matmul_dev(_ptr(y), _ptr(x), C.byref(t), n, d, stream), "gguf_matmul_dev")


def sync(stream=None) -> None:
    check(lib().vireo_sync(stream), "vireo_sync")


# ---------------------------------------------------------------------------
# MoE block (gguf_moe.h)
# ---------------------------------------------------------------------------

class MoeLayer:
    """One MoE FFN layer resident in HBM, evaluated by gguf_moe_ffn.

    ``layer`` is a ``vireo_b200.synth.MoeLayer`` or any object with ``spec``
    (dim, ffn_exp, n_experts, n_used, topk_renorm, *_type) and raw GGUF byte
    arrays ``router``, ``gate``, ``up``, ``down`` (experts outermost).
    Device memory is held in torch tensors (plumbing only)."""

    def __init__(self, layer, device: int = 0):
        import torch
        s = layer.spec
        self.spec = s
        self.device = torch.device("cuda", device)
        up = lambda a: torch.from_numpy(np.ascontiguousarray(a).view(np.uint8).reshape(-1)).to(self.device)
        self.router, self.gate, self.up, self.down = up(layer.router), up(layer.gate), up(layer.up), up(layer.down)
        self.desc = GgufMoeDesc(s.dim, s.ffn_exp, s.n_experts, s.n_used, s.topk_renorm, s.router_type,
                                s.gate_type, s.up_type, s.down_type, self.router.data_ptr(),
                                self.gate.data_ptr(), self.up.data_ptr(), self.down.data_ptr(),
                                self.gate.numel(), self.up.numel(), self.down.numel())
        h = C.c_void_p()
        check(lib().gguf_moe_create(C.byref(self.desc), C.byref(h)), "gguf_moe_create")
        self.h = h

    def ffn(self, hb, x, ids=None, wts=None, stream=None) -> None:
        """Device tensors: hb/x [n_tok, dim] fp32 (x updated), ids/wts [n_tok, n_used]."""
        n = hb.shape[0] if hb.dim() > 1 else 1
        check(lib().gguf_moe_ffn(self.h, hb.data_ptr(), x.data_ptr(), n,
                                 ids.data_ptr() if ids is not None else None,
                                 wts.data_ptr() if wts is not None else None, stream), "gguf_moe_ffn")

    def sync(self, stream=None) -> None:
        check(lib().gguf_moe_sync(self.h, stream), "gguf_moe_sync")

    def ffn_host(self, hb: np.ndarray, x: np.ndarray | None = None):
        """Host buffers through gguf_moe_ffn_host; returns (x_out, ids, wts)."""
        s = self.spec
        hb = np.ascontiguousarray(hb, dtype=np.float32).reshape(-1, s.dim)
        n = hb.shape[0]
        x = np.zeros_like(hb) if x is None else np.array(x, dtype=np.float32).reshape(n, s.dim)
        ids = np.zeros((n, s.n_used), dtype=np.int32)
        wts = np.zeros((n, s.n_used), dtype=np.float32)
        check(lib().gguf_moe_ffn_host(self.h, hb.ctypes.data, x.ctypes.data, n, ids.ctypes.data, wts.ctypes.data),
              "gguf_moe_ffn_host")
        return x, ids, wts

    def close(self) -> None:
        if getattr(self, "h", None):
            lib().gguf_moe_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def ep_place(expected_load, world: int) -> np.ndarray:
    """gguf_moe_ep_place: expert -> rank by expected load (host only)."""
    load = np.ascontiguousarray(expected_load, dtype=np.float64)
    owner = np.zeros(load.size, dtype=np.int32)
    check(lib().gguf_moe_ep_place(load.ctypes.data, load.size, world, owner.ctypes.data), "gguf_moe_ep_place")
    return owner


def ep_rows(counts, owner, rank: int):
    """gguf_moe_ep_rows (host only): (dst_off [n_experts], rows_here) for
    `rank` given the [world][n_experts] pair counts and the placement."""
    c = np.ascontiguousarray(counts, dtype=np.int32)
    o = np.ascontiguousarray(owner, dtype=np.int32)
    world, ne = c.shape
    off = np.zeros(ne, dtype=np.int32)
    here = C.c_int32()
    check(lib().gguf_moe_ep_rows(c.ctypes.data, o.ctypes.data, ne, world, rank, off.ctypes.data, C.byref(here)),
          "gguf_moe_ep_rows")
    return off, int(here.value)


def ep_unique_id() -> bytes:
    buf = C.create_string_buffer(128)
    check(lib().gguf_moe_ep_unique_id(buf), "gguf_moe_ep_unique_id")
    return buf.raw


class SharedExpert:
    """A shared expert (gguf_moe_shexp_*): ``sh`` is a
    ``vireo_b200.synth.SharedExpert`` (dim, ffn, *_type, raw GGUF ``gate``,
    ``up``, ``down`` and an optional fp32 ``gate_inp``)."""

    def __init__(self, sh, device: int = 0):
        import torch
        dev = torch.device("cuda", device)
        up = lambda a: torch.from_numpy(np.ascontiguousarray(a).view(np.uint8).reshape(-1)).to(dev)
        self._keep = [up(sh.gate), up(sh.up), up(sh.down)]
        gi = None
        if sh.gate_inp is not None:
            gi = torch.from_numpy(np.ascontiguousarray(sh.gate_inp, dtype=np.float32)).to(dev)
            self._keep.append(gi)
        g, u, dn = self._keep[:3]
        self.desc = GgufMoeShexpDesc(sh.dim, sh.ffn, sh.gate_type, sh.up_type, sh.down_type, g.data_ptr(),
                                     u.data_ptr(), dn.data_ptr(), gi.data_ptr() if gi is not None else None)
        h = C.c_void_p()
        check(lib().gguf_moe_shexp_create(C.byref(self.desc), C.byref(h)), "gguf_moe_shexp_create")
        self.h = h

    def ffn(self, hb, x, stream=None) -> None:
        n = hb.shape[0] if hb.dim() > 1 else 1
        check(lib().gguf_moe_shexp_ffn(self.h, hb.data_ptr(), x.data_ptr(), n, stream), "gguf_moe_shexp_ffn")

    def sync(self, stream=None) -> None:
        check(lib().gguf_moe_shexp_sync(self.h, stream), "gguf_moe_shexp_sync")

    def close(self) -> None:
        if self.h:
            lib().gguf_moe_shexp_destroy(self.h)
            self.h = None


class MoeLayerEP:
    """One rank's share of an expert-parallel MoE layer (gguf_moe_ep_*).
    Every rank constructs it with the same owner table and unique id."""

    def __init__(self, layer, owner, rank: int, world: int, uid: bytes, max_tokens: int, device: int = 0):
        import torch
        s = layer.spec
        self.spec = s
        dev = torch.device("cuda", device)
        up = lambda a: torch.from_numpy(np.ascontiguousarray(a).view(np.uint8).reshape(-1)).to(dev)
        self._keep = [up(layer.router), up(layer.gate), up(layer.up), up(layer.down)]
        r, g, u, dn = self._keep
        self.desc = GgufMoeDesc(s.dim, s.ffn_exp, s.n_experts, s.n_used, s.topk_renorm, s.router_type,
                                s.gate_type, s.up_type, s.down_type, r.data_ptr(), g.data_ptr(), u.data_ptr(),
                                dn.data_ptr(), g.numel(), u.numel(), dn.numel())
        self.owner = np.ascontiguousarray(owner, dtype=np.int32)
        buf = C.create_string_buffer(uid, 128)
        h = C.c_void_p()
        check(lib().gguf_moe_ep_create(C.byref(self.desc), self.owner.ctypes.data, rank, world, max_tokens, buf,
                                       C.byref(h)), "gguf_moe_ep_create")
        self.h = h

    def prefill(self, hb_bf16, x, bias=None, ids=None, wts=None, stream=None) -> None:
        n = hb_bf16.shape[0]
        check(lib().gguf_moe_prefill_ep(self.h, hb_bf16.data_ptr(), x.data_ptr(), n,
                                        bias.data_ptr() if bias is not None else None,
                                        ids.data_ptr() if ids is not None else None,
                                        wts.data_ptr() if wts is not None else None, stream), "gguf_moe_prefill_ep")

    def sync(self, stream=None) -> None:
        check(lib().gguf_moe_ep_sync(self.h, stream), "gguf_moe_ep_sync")

    def close(self) -> None:
        if getattr(self, "h", None):
            lib().gguf_moe_ep_destroy(self.h)
            self.h = None


class GgufDecoderDesc(C.Structure):
    _fields_ = [("n_layers", C.c_int), ("dim", C.c_int), ("n_heads", C.c_int), ("n_kv_heads", C.c_int),
                ("head_size", C.c_int), ("vocab", C.c_int), ("eps", C.c_float), ("rope_base", C.c_float),
                ("max_ctx", C.c_int), ("kv_f16", C.c_int), ("tok_embd_type", C.c_uint32), ("tok_embd", C.c_void_p),
                ("out_norm", C.c_void_p), ("lm_head_type", C.c_uint32), ("lm_head", C.c_void_p)]


class GgufDecoderLayer(C.Structure):
    _fields_ = [("attn_norm", C.c_void_p), ("ffn_norm", C.c_void_p), ("wq_type", C.c_uint32),
                ("wk_type", C.c_uint32), ("wv_type", C.c_uint32), ("wo_type", C.c_uint32), ("wq", C.c_void_p),
                ("wk", C.c_void_p), ("wv", C.c_void_p), ("wo", C.c_void_p), ("bq", C.c_void_p), ("bk", C.c_void_p),
                ("bv", C.c_void_p), ("q_norm", C.c_void_p), ("k_norm", C.c_void_p), ("q_norm_len", C.c_int),
                ("k_norm_len", C.c_int), ("moe", C.c_void_p)]


def _decoder_api(L):
    if getattr(L, "_decoder_api", False):
        return
    L.gguf_decoder_create.argtypes = [C.POINTER(GgufDecoderDesc), C.c_void_p, C.POINTER(C.c_void_p)]
    L.gguf_decoder_step.argtypes = [C.c_void_p, C.c_int, C.c_int, C.c_void_p, C.c_void_p, C.c_void_p]
    L.gguf_decoder_step_dev.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, C.c_void_p, C.c_void_p]
    L.gguf_decoder_hidden.argtypes = [C.c_void_p]
    L.gguf_decoder_hidden.restype = C.c_void_p
    L.gguf_decoder_sync.argtypes = [C.c_void_p, C.c_void_p]
    L.gguf_decoder_destroy.argtypes = [C.c_void_p]
    L.gguf_decoder_destroy.restype = None
    L._decoder_api = True


class Decoder:
    """A whole MoE decoder on the device (gguf_decoder_*): the reference's
    forward() (src/gguf_run.c:216-252) one step per call.  ``dec`` is a
    ``vireo_b200.synth.Decoder`` (or any object with the same fields).  Each
    layer gets its own device copy of its tensors, also when the generated
    layers repeat, so no step reads another layer's bytes out of L2."""

    def __init__(self, dec, max_ctx: int, kv_f16: bool = True, device: int = 0):
        import torch
        L = lib()
        _decoder_api(L)
        s = dec.spec
        self.spec = s
        dev = torch.device("cuda", device)
        self.device = dev
        uploaded = {}

        def up(a):
            """a device copy per call (distinct addresses), uploaded once per host array"""
            if a is None:
                return None
            key = id(a)
            if key not in uploaded:
                uploaded[key] = torch.from_numpy(np.ascontiguousarray(a).view(np.uint8).reshape(-1)).to(dev)
                return uploaded[key]
            return uploaded[key].clone()

        self._keep = []
        keep = self._keep.append
        ptr = lambda t: t.data_ptr() if t is not None else None
        tok, on, lm = up(dec.tok_embd), up(dec.out_norm), up(dec.lm_head)
        keep(tok), keep(on), keep(lm)
        self.desc = GgufDecoderDesc(s.n_layers, s.dim, s.n_heads, s.n_kv_heads, s.head_size, s.vocab, s.eps,
                                    s.rope_base, max_ctx, int(kv_f16), s.embd_type, ptr(tok), ptr(on), s.lm_type,
                                    ptr(lm))
        self.moe = []
        rows = []
        for ly in dec.layers:
            t = [up(a) for a in (ly.attn_norm, ly.ffn_norm, ly.wq, ly.wk, ly.wv, ly.wo, ly.q_norm, ly.k_norm)]
            for x in t:
                keep(x)
            m = _DeviceMoe(ly.moe, up)
            self.moe.append(m)
            qn = s.head_size if s.qk_norm == "head" else s.q_dim
            kn = s.head_size if s.qk_norm == "head" else s.kv_dim
            rows.append(GgufDecoderLayer(ptr(t[0]), ptr(t[1]), s.attn_type, s.attn_type, s.attn_type, s.attn_type,
                                         ptr(t[2]), ptr(t[3]), ptr(t[4]), ptr(t[5]), None, None, None, ptr(t[6]),
                                         ptr(t[7]), qn if t[6] is not None else 0, kn if t[7] is not None else 0,
                                         m.h))
        self.layers = (GgufDecoderLayer * len(rows))(*rows)
        h = C.c_void_p()
        check(L.gguf_decoder_create(C.byref(self.desc), self.layers, C.byref(h)), "gguf_decoder_create")
        self.h = h

    def step(self, token: int, pos: int, logits=None, next=None, stream=None) -> None:
        """Device tensors logits [vocab] fp32 / next [1] int32, or None."""
        check(lib().gguf_decoder_step(self.h, int(token), int(pos), logits.data_ptr() if logits is not None else None,
                                      next.data_ptr() if next is not None else None, stream), "gguf_decoder_step")

    def step_dev(self, token, pos: int, logits=None, next=None, stream=None) -> None:
        """token: device int32 tensor [1] (e.g. the previous step's next)."""
        check(lib().gguf_decoder_step_dev(self.h, token.data_ptr(), int(pos),
                                          logits.data_ptr() if logits is not None else None,
                                          next.data_ptr() if next is not None else None, stream),
              "gguf_decoder_step_dev")

    def sync(self, stream=None) -> None:
        check(lib().gguf_decoder_sync(self.h, stream), "gguf_decoder_sync")

    def close(self) -> None:
        if getattr(self, "h", None):
            lib().gguf_decoder_destroy(self.h)
            self.h = None
        for m in getattr(self, "moe", []):
            m.close()
        self.moe = []

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class _DeviceMoe:
    """A gguf_moe handle over device copies made by `up` (Decoder's uploader)."""

    def __init__(self, layer, up):
        s = layer.spec
        self.spec = s
        self.router, self.gate, self.up, self.down = up(layer.router), up(layer.gate), up(layer.up), up(layer.down)
        self.desc = GgufMoeDesc(s.dim, s.ffn_exp, s.n_experts, s.n_used, s.topk_renorm, s.router_type,
                                s.gate_type, s.up_type, s.down_type, self.router.data_ptr(),
                                self.gate.data_ptr(), self.up.data_ptr(), self.down.data_ptr(),
                                self.gate.numel(), self.up.numel(), self.down.numel())
        h = C.c_void_p()
        check(lib().gguf_moe_create(C.byref(self.desc), C.byref(h)), "gguf_moe_create")
        self.h = h

    def close(self):
        if getattr(self, "h", None):
            lib().gguf_moe_destroy(self.h)
            self.h = None


# ---------------------------------------------------------------------------
# paged key-value pool (gguf_kv.h)
# ---------------------------------------------------------------------------

class GgufKvDesc(C.Structure):
    _fields_ = [("n_heads", C.c_int), ("n_kv_heads", C.c_int), ("head_size", C.c_int), ("page_size", C.c_int),
                ("n_pages", C.c_int), ("kv_type", C.c_uint32), ("act_type", C.c_uint32), ("k", C.c_void_p),
                ("v", C.c_void_p), ("page_stride", C.c_int64), ("head_stride", C.c_int64), ("pos_stride", C.c_int64),
                ("eps", C.c_float), ("rope_base", C.c_float), ("rope_dim", C.c_int)]


class GgufKvPlanArgs(C.Structure):
    _fields_ = [("n_seqs", C.c_int), ("page_size", C.c_int), ("n_pages", C.c_int), ("max_pages", C.c_int),
                ("n_slots", C.c_int), ("table_stride", C.c_int64), ("past", C.c_void_p), ("add", C.c_void_p),
                ("table", C.c_void_p), ("ring", C.c_void_p), ("state", C.c_void_p), ("slots", C.c_void_p),
                ("pos", C.c_void_p), ("cu", C.c_void_p), ("kv_len", C.c_void_p), ("granted", C.c_void_p),
                ("state_out", C.c_void_p)]


class GgufKvAppendArgs(C.Structure):
    _fields_ = [("n_tokens", C.c_int), ("q", C.c_void_p), ("k", C.c_void_p), ("v", C.c_void_p),
                ("q_stride", C.c_int64), ("k_stride", C.c_int64), ("v_stride", C.c_int64), ("q_out", C.c_void_p),
                ("q_out_stride", C.c_int64), ("pos", C.c_void_p), ("slots", C.c_void_p), ("bq", C.c_void_p),
                ("bk", C.c_void_p), ("bv", C.c_void_p), ("q_norm", C.c_void_p), ("k_norm", C.c_void_p),
                ("q_norm_len", C.c_int), ("k_norm_len", C.c_int), ("means", C.c_void_p)]


class GgufKvAttnArgs(C.Structure):
    _fields_ = [("n_seqs", C.c_int), ("max_pages", C.c_int), ("q", C.c_void_p), ("q_stride", C.c_int64),
                ("out", C.c_void_p), ("out_stride", C.c_int64), ("table", C.c_void_p), ("table_stride", C.c_int64),
                ("kv_len", C.c_void_p), ("scale", C.c_float), ("ws", C.c_void_p), ("ws_bytes", C.c_size_t)]


class GgufKvSelectArgs(C.Structure):
    _fields_ = [("means", C.c_void_p), ("n_sink", C.c_int), ("n_window", C.c_int), ("n_top", C.c_int),
                ("sel", C.c_void_p)]


# The same layouts for struct.pack: a call's arguments are packed in a fifth of
# the time that filling a ctypes structure takes.
_PLAN_PACK = struct.Struct("@5iq11P").pack
_APPEND_PACK = struct.Struct("@i3P3qPq7P2iP").pack
_ATTN_PACK = struct.Struct("@2iPqPqPqPfPN").pack
_SELECT_PACK = struct.Struct("@P3iP").pack


def _kv_api():
    L = lib()
    if not getattr(L, "_kv_api", False):
        L.gguf_kv_create.argtypes = [C.POINTER(GgufKvDesc), C.POINTER(C.c_void_p)]
        L.gguf_kv_destroy.argtypes = [C.c_void_p]
        L.gguf_kv_destroy.restype = None
        L.gguf_kv_sync.argtypes = [C.c_void_p, C.c_void_p]
        # argument structures: by reference, or packed as bytes
        L.gguf_kv_plan.argtypes = [C.c_void_p, C.c_void_p]
        L.gguf_kv_append.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p]
        L.gguf_kv_attn.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p]
        L.gguf_kv_attn_topk.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p]
        L.gguf_kv_workspace.argtypes = [C.c_void_p, C.c_int, C.c_int, C.c_int]
        L.gguf_kv_workspace.restype = C.c_size_t
        L._kv_api = True
    return L


def _need(ok, what: str) -> None:
    if not ok:
        raise VireoError(-1, what)


_kv_dev = None  # the library's device, once a call has had tensors on it


def _kv_device(dev: int) -> None:
    """The library works on one device: this one from now on, or an error if it has another."""
    global _kv_dev
    if dev != _kv_dev:
        import torch
        current = torch.cuda.current_device()
        try:
            check(lib().vireo_device_init(dev), f"cuda:{dev} is not the library's device")
        finally:
            torch.cuda.set_device(current)
        _kv_dev = dev


# The helpers below run a dozen times per call of a few microseconds: the
# message is made only when a check fails, devices are compared by index and
# each property of a tensor is asked for once.

def _kv_pack(pack, *values) -> bytes:
    try:
        return pack(*values)
    except (struct.error, OverflowError) as e:
        raise VireoError(-1, f"an argument does not fit its type: {e}") from None


def _kv_ptr(t, n: int, dtype, dev: int, name: str) -> int:
    """The address of a contiguous tensor of n values of this type on device dev."""
    if t.numel() != n or t.dtype is not dtype or t.get_device() != dev or not t.is_contiguous():
        raise VireoError(-1, f"{name}: {n} contiguous {dtype} values on cuda:{dev} are needed")
    return t.data_ptr()


def _kv_rows(t, n: int, width: int, dtype, dev: int, name: str):
    """(address, row stride) of n rows of `width` contiguous elements: [n, width] or [n, heads, size]."""
    shape, stride = t.shape, t.stride()
    if len(shape) == 2:
        ok = shape[1] == width and (stride[1] == 1 or width == 1)
    else:
        ok = (len(shape) == 3 and shape[1] * shape[2] == width and stride[2] == 1
              and (shape[1] == 1 or stride[1] == shape[2]))
    if not ok or shape[0] != n or t.dtype is not dtype or t.get_device() != dev:
        raise VireoError(-1, f"{name}: {n} rows of {width} contiguous {dtype} values on cuda:{dev} are needed")
    return t.data_ptr(), (stride[0] if n > 1 else width)


def _kv_table(t, n: int, dtype, dev: int):
    """(address, row stride, width) of a block table [n, max_pages]."""
    shape = t.shape
    if len(shape) == 2 and shape[0] == n and shape[1] > 0 and t.dtype is dtype and t.get_device() == dev:
        stride = t.stride()
        if stride[1] == 1 or shape[1] == 1:
            return t.data_ptr(), (stride[0] if n > 1 else shape[1]), shape[1]
    raise VireoError(-1, f"table: [{n}, max_pages] {dtype} rows on cuda:{dev} are needed")


def _kv_stream(dev: int, stream) -> int:
    """The raw stream of a call: the given one, or torch's current stream on
    the device (the legacy default stream by its own handle, since 0 stands for
    the library's stream)."""
    if stream is None:
        import torch
        return torch._C._cuda_getCurrentRawStream(dev) or 1
    return getattr(stream, "cuda_stream", stream) or 1


def kv_plan(past, add, table, ring, state, page_size: int, *, slots, pos, cu, kv_len, granted, state_out,
            stream=None) -> None:
    """gguf_kv_plan: block tables, slots and positions from request lengths.

    past, add [n] int32; table [n, max_pages] int32 (written where pages are
    added); ring [n_pages] and state [2] = (head, count) int32: the free
    pages; slots [n_slots] int64 and pos [n_slots] int32, cu [n + 1], kv_len
    [n], granted [n], state_out [2] int32: written.  kv_len may be past and
    state_out may be state.  stream: a raw handle or a torch stream; torch's
    current stream by default."""
    import torch
    dev, i32, n, n_pages, n_slots = past.get_device(), torch.int32, past.numel(), ring.numel(), slots.numel()
    if dev < 0:
        raise VireoError(-1, "kv_plan: CUDA tensors are needed")
    if dev != _kv_dev:
        _kv_device(dev)
    tp, ts, width = _kv_table(table, n, i32, dev)
    a = _kv_pack(_PLAN_PACK, n, page_size, n_pages, width, n_slots, ts, _kv_ptr(past, n, i32, dev, "past"),
                 _kv_ptr(add, n, i32, dev, "add"), tp, _kv_ptr(ring, n_pages, i32, dev, "ring"),
                 _kv_ptr(state, 2, i32, dev, "state"), _kv_ptr(slots, n_slots, torch.int64, dev, "slots"),
                 _kv_ptr(pos, n_slots, i32, dev, "pos"), _kv_ptr(cu, n + 1, i32, dev, "cu"),
                 _kv_ptr(kv_len, n, i32, dev, "kv_len"), _kv_ptr(granted, n, i32, dev, "granted"),
                 _kv_ptr(state_out, 2, i32, dev, "state_out"))
    check(_kv_api().gguf_kv_plan(a, _kv_stream(dev, stream)), "gguf_kv_plan")


class PagedKV:
    """One layer's paged key-value pool (gguf_kv_*).

    k, v: torch CUDA tensors seen as [n_pages, n_kv_heads, page_size,
    head_size] with the same strides and the last one 1 (a pool with positions
    outside heads is passed as ``pool.transpose(1, 2)``); they stay the
    caller's.  act_dtype: of queries, new keys and values and outputs (the
    cache's by default; float32 also goes with a float16 cache).  Every call
    runs on `stream` (a raw handle or a torch stream), torch's current one by
    default, and may be captured into a CUDA graph; the attention's
    workspace comes from torch's allocator per call, on that stream.  Tensors
    are not recorded on a stream passed as `stream`: keep them until it has
    done with them, as with any stream that torch does not know of."""

    def __init__(self, k, v, n_heads: int, act_dtype=None, eps: float = 1e-6, rope_base: float = 10000.0,
                 rope_dim: int | None = None):
        import torch
        self.h = None
        types = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}
        L = _kv_api()
        act_dtype = k.dtype if act_dtype is None else act_dtype
        _need(k.dim() == 4 and k.shape == v.shape and k.stride() == v.stride() and k.stride(3) == 1
              and k.dtype == v.dtype and k.device == v.device and k.device.type == "cuda",
              "k, v: [pages, kv heads, positions, size] CUDA tensors of one type and layout are needed")
        _need(k.dtype in types and act_dtype in types, "types: float32, float16 and bfloat16 only")
        self.k, self.v, self.device = k, v, k.get_device()
        _kv_device(self.device)
        self.n_pages, self.n_kv_heads, self.page_size, self.head_size = k.shape
        self.n_heads, self.kv_dtype, self.act_dtype = int(n_heads), k.dtype, act_dtype
        self.desc = GgufKvDesc(self.n_heads, self.n_kv_heads, self.head_size, self.page_size, self.n_pages,
                               types[k.dtype], types[act_dtype], k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1),
                               k.stride(2), eps, rope_base, self.head_size if rope_dim is None else rope_dim)
        h = C.c_void_p()
        check(L.gguf_kv_create(C.byref(self.desc), C.byref(h)), "gguf_kv_create")
        self.h = h
        self._qw, self._kw = self.n_heads * self.head_size, self.n_kv_heads * self.head_size
        self._lib, self._ws_bytes = L, {}

    def append(self, q, k, v, pos, slots, q_out, *, q_norm=None, k_norm=None, bq=None, bk=None, bv=None, means=None,
               stream=None) -> None:
        """gguf_kv_append: q, k, v [n, heads * size] (or [n, heads, size]) rows
        of act_dtype, pos [n] int32, slots [n] int64; writes q_out, the pool
        and, given, means [n_pages, n_kv_heads, size] of the cache's type."""
        import torch
        n, dev, f32, qw, kw, a = pos.numel(), self.device, torch.float32, self._qw, self._kw, self.act_dtype
        qp, qs = _kv_rows(q, n, qw, a, dev, "q")
        kp, ks = _kv_rows(k, n, kw, a, dev, "k")
        vp, vs = _kv_rows(v, n, kw, a, dev, "v")
        op, os_ = _kv_rows(q_out, n, qw, a, dev, "q_out")
        nq, nk = 0 if q_norm is None else q_norm.numel(), 0 if k_norm is None else k_norm.numel()
        if (nq == 0) != (q_norm is None) or (nk == 0) != (k_norm is None):
            raise VireoError(-1, "q_norm, k_norm: empty")
        args = _APPEND_PACK(n, qp, kp, vp, qs, ks, vs, op, os_, _kv_ptr(pos, n, torch.int32, dev, "pos"),
                            _kv_ptr(slots, n, torch.int64, dev, "slots"),
                            0 if bq is None else _kv_ptr(bq, qw, f32, dev, "bq"),
                            0 if bk is None else _kv_ptr(bk, kw, f32, dev, "bk"),
                            0 if bv is None else _kv_ptr(bv, kw, f32, dev, "bv"),
                            0 if nq == 0 else _kv_ptr(q_norm, nq, f32, dev, "q_norm"),
                            0 if nk == 0 else _kv_ptr(k_norm, nk, f32, dev, "k_norm"), nq, nk,
                            0 if means is None else _kv_ptr(means, self.n_pages * kw, self.kv_dtype, dev, "means"))
        check(self._lib.gguf_kv_append(self.h, args, _kv_stream(dev, stream)), "gguf_kv_append")

    def _attn_args(self, q, table, kv_len, out, scale, n_select, stream):
        """(gguf_kv_attn_args, packed; requests; the workspace that it points to)."""
        import torch
        n, dev, w, a = kv_len.numel(), self.device, self._qw, self.act_dtype
        qp, qs = _kv_rows(q, n, w, a, dev, "q")
        op, os_ = _kv_rows(out, n, w, a, dev, "out")
        tp, ts, width = _kv_table(table, n, torch.int32, dev)
        nbytes = self._ws_bytes.get((n, width, n_select))
        if nbytes is None:
            if len(self._ws_bytes) >= 256:
                self._ws_bytes.clear()
            nbytes = self._ws_bytes[n, width, n_select] = self._lib.gguf_kv_workspace(self.h, n, width, n_select)
        if stream is None:
            ws = q.new_empty(nbytes, dtype=torch.uint8)
        else:  # memory of the stream that uses it
            raw = _kv_stream(dev, stream)
            with torch.cuda.stream(torch.cuda.ExternalStream(raw, device=dev) if raw != 1
                                   else torch.cuda.default_stream(dev)):
                ws = q.new_empty(nbytes, dtype=torch.uint8)
        return _kv_pack(_ATTN_PACK, n, width, qp, qs, op, os_, tp, ts, _kv_ptr(kv_len, n, torch.int32, dev, "kv_len"),
                        0.0 if scale is None else scale, ws.data_ptr(), nbytes), n, ws

    def attn(self, q, table, kv_len, out, scale=None, stream=None) -> None:
        """gguf_kv_attn: q, out [n, n_heads * size] (or [n, n_heads, size]),
        table [n, max_pages] int32, kv_len [n] int32; scale 1 / sqrt(size) by
        default, and where it is 0."""
        args, _, ws = self._attn_args(q, table, kv_len, out, scale, 0, stream)
        check(self._lib.gguf_kv_attn(self.h, args, _kv_stream(self.device, stream)), "gguf_kv_attn")

    def attn_topk(self, q, table, kv_len, means, n_sink: int, n_window: int, n_top: int, out, sel=None, scale=None,
                  stream=None) -> None:
        """gguf_kv_attn_topk: attention over each request's first n_sink, last
        n_window and n_top best pages; sel, given, receives their indices
        [n, n_kv_heads, n_sink + n_window + n_top] int32."""
        import torch
        ns = n_sink + n_window + n_top
        if n_sink < 0 or n_window < 1 or n_top < 0 or ns >= 2 ** 21:
            raise VireoError(-1, "n_sink >= 0, n_window >= 1 and n_top >= 0, together below 2^21, are needed")
        args, n, ws = self._attn_args(q, table, kv_len, out, scale, ns, stream)
        dev = self.device
        sp = 0 if sel is None else _kv_ptr(sel, n * self.n_kv_heads * ns, torch.int32, dev, "sel")
        s = _kv_pack(_SELECT_PACK, _kv_ptr(means, self.n_pages * self._kw, self.kv_dtype, dev, "means"), n_sink,
                     n_window, n_top, sp)
        check(self._lib.gguf_kv_attn_topk(self.h, args, s, _kv_stream(dev, stream)), "gguf_kv_attn_topk")

    def sync(self, stream=None) -> None:
        """Waits for the stream; raises what the device reported."""
        check(self._lib.gguf_kv_sync(self.h, _kv_stream(self.device, stream)), "gguf_kv_sync")

    def close(self) -> None:
        if getattr(self, "h", None):
            lib().gguf_kv_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
