"""Python front end of libobsmoe.so (include/obs_moe.h) for the B200 MoE path.

Mirrors the reference's MoE helpers in src/forward.rs and src/router.rs by name
and argument meaning: ``gate_gpu`` (forward.rs:386-397), ``route``
(router.rs:25-56), ``dispatch`` (the grouping of forward.rs:203-216),
``expert_ffn`` (dequant/matmul_raw + swiglu, forward.rs:303-321,370-375),
``moe_forward`` (the MoE section of forward_layer / prefill_batched).  Errors
raise ``ObsError`` carrying the library's message, the way the reference's
helpers return ``Err(String)``.

Device buffers are passed as raw pointers: any object with ``data_ptr()``
(a torch CUDA tensor, used here only as device-memory plumbing) or an int.
There is no CPU fallback: if the CUDA library is missing this module raises.
"""
from __future__ import annotations

import ctypes as C
import os
from dataclasses import dataclass

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libobsmoe.so")

OBS_OK = 0
PATH_AUTO, PATH_DECODE, PATH_PREFILL = 0, 1, 2
_STATUS = {1: "INVALID", 2: "CUDA", 3: "NOMEM", 4: "STATE", 5: "TIMEOUT", 6: "NCCL", 7: "UNSUPPORTED"}

# every entry point include/obs_moe.h declares
EXPORTS = (
    "obs_abi_version", "obs_create", "obs_destroy", "obs_last_error", "obs_memory_bytes",
    "obs_load_layer", "obs_synth_layer", "obs_synth_activations", "obs_moe_forward",
    "obs_moe_forward_host", "obs_moe_forward_host_async", "obs_moe_host_join", "obs_gate", "obs_route", "obs_dispatch", "obs_expert_ffn",
    "obs_expert_gemm_f32", "obs_check_device", "obs_profile_enable", "obs_profile_read",
    "obs_trace_enable", "obs_decode_ffn_static", "obs_kernel_launches", "obs_ep_handle", "obs_ep_connect",
    "obs_rmsnorm", "obs_moe_stack_forward", "obs_set_wait_limit", "obs_probe_wait", "obs_struct_layout",
    "obs_load_layer_safetensors", "obs_expert_file_info", "obs_load_head", "obs_embed", "obs_lm_head",
    "obs_attn_init", "obs_load_attn", "obs_attn_forward", "obs_kv_read", "obs_debug_gemm_tiles",
    "obs_ep_set_placement", "obs_ep_get_placement", "obs_ep_plan_placement",
    "obs_paged_init", "obs_paged_append", "obs_paged_decode", "obs_paged_prefill", "obs_paged_evict",
    "obs_paged_attn_forward", "obs_paged_struct_layout",
)
EP_HANDLE_BYTES = 64
STAGES = ("router", "topk", "dispatch", "gemm_gateup", "gemm_down", "combine", "decode_gateup", "decode_down",
          "decode_fused", "ep_send", "ep_recv", "ep_return")


class ObsError(RuntimeError):
    def __init__(self, status: int, msg: str):
        super().__init__(f"obs {_STATUS.get(status, status)}: {msg}")
        self.status = status


class Config(C.Structure):
    _fields_ = [("hidden", C.c_int32), ("inter", C.c_int32), ("n_experts", C.c_int32),
                ("top_k", C.c_int32), ("group_size", C.c_int32), ("n_layers", C.c_int32),
                ("max_tokens", C.c_int32), ("norm_topk", C.c_int32),
                ("decode_max_tokens", C.c_int32), ("rms_eps", C.c_float),
                ("ep_world", C.c_int32), ("ep_rank", C.c_int32)]


class HeadWeights(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("embed_w", "embed_s", "embed_b", "lm_w", "lm_s", "lm_b", "norm_w")]


class AttnWeights(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in (
        "q_w", "q_s", "q_b", "k_w", "k_s", "k_b", "v_w", "v_s", "v_b", "o_w", "o_s", "o_b",
        "in_norm", "q_norm", "k_norm")]


class AttnConfig(C.Structure):
    _fields_ = [("n_heads", C.c_int32), ("n_kv_heads", C.c_int32), ("head_dim", C.c_int32),
                ("max_seq", C.c_int32), ("n_seqs", C.c_int32), ("rope_theta", C.c_float)]


class LayerWeights(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in (
        "router_w", "router_s", "router_b", "gate_w", "gate_s", "gate_b",
        "up_w", "up_s", "up_b", "down_w", "down_s", "down_b")]


class PagedConfig(C.Structure):
    _fields_ = [(n, C.c_int32) for n in (
        "n_heads", "n_kv_heads", "head_dim", "page_size", "max_seqs", "max_kv_len", "dtype", "weights")]


class PagedView(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("block_table", C.c_void_p), ("kv_len", C.c_void_p),
                ("page_stride", C.c_int64), ("slot_stride", C.c_int64), ("head_stride", C.c_int64),
                ("n_seqs", C.c_int32), ("n_pages", C.c_int32), ("table_stride", C.c_int32), ("table_pages", C.c_int32)]


DTYPE_BF16, DTYPE_F16 = 0, 1
_PLANS = {}  # one tuple for equal (page_size, n_kv_heads, head_dim, dtype): calls compare them by identity
_DTYPES = {"bf16": DTYPE_BF16, "f16": DTYPE_F16}


class PagedKV:
    """One layer's paged key/value cache (obs_paged_kv) over tensors the caller owns: k and v
    [n_pages, page_size, n_kv_heads, head_dim] of 16-bit elements (any strides, head_dim
    consecutive), block_table int32 [n_seqs, pages], kv_len int32 [n_seqs], all on the GPU.
    Keeps the tensors alive; their contents may change between calls."""

    def __init__(self, k, v, block_table, kv_len):
        for name, t in (("k", k), ("v", v)):
            if t.dim() != 4 or t.element_size() != 2 or (t.shape[3] > 1 and t.stride(3) != 1):
                raise ValueError(f"{name}: [n_pages, page_size, n_kv_heads, head_dim] of 16-bit elements, the last consecutive")
        if v.shape != k.shape or v.stride() != k.stride() or v.dtype != k.dtype:
            raise ValueError("k and v must have one shape, one type and the same strides")
        if block_table.dim() != 2 or block_table.element_size() != 4 or block_table.is_floating_point():
            raise ValueError("block_table: int32 [n_seqs, pages]")
        if block_table.shape[1] > 1 and block_table.stride(1) != 1:
            raise ValueError("block_table's rows must be consecutive")
        if kv_len.dim() != 1 or kv_len.element_size() != 4 or kv_len.is_floating_point() or not kv_len.is_contiguous():
            raise ValueError("kv_len: consecutive int32 [n_seqs]")
        if kv_len.shape[0] != block_table.shape[0]:
            raise ValueError("kv_len and block_table have different numbers of sequences")
        if block_table.shape[0] > 1 and block_table.stride(0) < block_table.shape[1]:
            raise ValueError("block_table's rows may not overlap")
        if not (k.is_cuda and v.is_cuda and block_table.is_cuda and kv_len.is_cuda):
            raise ValueError("k, v, block_table and kv_len must be on the GPU")
        self.tensors = (k, v, block_table, kv_len)
        self.i32 = kv_len.dtype
        self.dtype, self.kv_shape = k.dtype, tuple(k.shape[1:])  # kv_shape: page_size, n_kv_heads, head_dim
        plan = (*self.kv_shape, "bf16" if "bfloat16" in str(k.dtype) else "f16")
        self.plan = _PLANS.setdefault(plan, plan)
        self.n_seqs = block_table.shape[0]
        self.view = PagedView(k.data_ptr(), v.data_ptr(), block_table.data_ptr(), kv_len.data_ptr(),
                              k.stride(0), k.stride(1), k.stride(2), self.n_seqs, k.shape[0],
                              block_table.stride(0), block_table.shape[1])
        self.ref = C.byref(self.view)


_LIB = None


def lib() -> C.CDLL:
    """Load libobsmoe.so (built by project-obsidian_b200/build.py)."""
    global _LIB
    if _LIB is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"{LIB_PATH} is missing: build it with python project-obsidian_b200/build.py")
        L = C.CDLL(LIB_PATH)
        vp, i32, i64 = C.c_void_p, C.c_int, C.c_uint64
        L.obs_abi_version.restype = i32
        L.obs_create.argtypes = [C.POINTER(Config), i32, C.POINTER(vp)]
        L.obs_destroy.argtypes = [vp]
        L.obs_last_error.restype = C.c_char_p
        L.obs_last_error.argtypes = [vp]
        L.obs_memory_bytes.argtypes = [vp, C.POINTER(C.c_size_t), C.POINTER(C.c_size_t)]
        L.obs_load_layer.argtypes = [vp, i32, C.POINTER(LayerWeights), i32]
        L.obs_synth_layer.argtypes = [vp, i32, i64]
        L.obs_synth_activations.argtypes = [i64, C.c_uint32, i32, i32, i32, C.c_float, vp, vp]
        L.obs_moe_forward.argtypes = [vp, i32, vp, vp, vp, i32, vp, i32, vp]
        L.obs_moe_forward_host.argtypes = [vp, i32, vp, vp, vp, i32, vp, i32, vp]
        L.obs_moe_forward_host_async.argtypes = [vp, i32, vp, vp, vp, i32, vp, i32, vp]
        L.obs_moe_host_join.argtypes = [vp, vp]
        L.obs_gate.argtypes = [vp, i32, vp, vp, i32, vp]
        L.obs_route.argtypes = [vp, vp, vp, i32, vp, vp, vp]
        L.obs_dispatch.argtypes = [vp, vp, i32, vp, vp, vp, vp]
        L.obs_expert_ffn.argtypes = [vp, i32, vp, vp, i32, i32, vp, vp]
        L.obs_expert_gemm_f32.argtypes = [vp, i32, i32, i32, vp, i32, vp, vp]
        L.obs_check_device.argtypes = [vp, vp]
        L.obs_profile_enable.argtypes = [vp, i32]
        L.obs_profile_read.argtypes = [vp, C.POINTER(C.c_float), C.POINTER(C.c_int32)]
        L.obs_trace_enable.argtypes = [vp, vp, i32]
        L.obs_kernel_launches.argtypes = [C.POINTER(C.c_uint64)]
        L.obs_ep_handle.argtypes = [vp, vp]
        L.obs_ep_connect.argtypes = [vp, vp]
        L.obs_ep_set_placement.argtypes = [vp, i32, C.POINTER(C.c_int32)]
        L.obs_ep_get_placement.argtypes = [vp, i32, C.POINTER(C.c_int32)]
        L.obs_ep_plan_placement.argtypes = [C.POINTER(C.c_int64), i32, i32, C.POINTER(C.c_int32)]
        L.obs_rmsnorm.argtypes = [vp, vp, vp, i32, vp, vp]
        L.obs_moe_stack_forward.argtypes = [vp, i32, i32, vp, i32, vp, i32, vp]
        L.obs_load_layer_safetensors.argtypes = [vp, i32, C.c_char_p, vp, vp, vp]
        L.obs_expert_file_info.argtypes = [C.c_char_p, C.POINTER(C.c_int32), C.POINTER(C.c_int32),
                                           C.POINTER(C.c_int32)]
        L.obs_load_head.argtypes = [vp, i32, C.POINTER(HeadWeights), i32]
        L.obs_embed.argtypes = [vp, vp, i32, vp, vp]
        L.obs_lm_head.argtypes = [vp, vp, i32, vp, vp, vp]
        L.obs_debug_gemm_tiles.argtypes = [vp, i32, vp, i32, vp]
        L.obs_attn_init.argtypes = [vp, C.POINTER(AttnConfig)]
        L.obs_load_attn.argtypes = [vp, i32, C.POINTER(AttnWeights), i32]
        L.obs_attn_forward.argtypes = [vp, i32, vp, vp, i32, vp, vp, vp]
        L.obs_kv_read.argtypes = [vp, i32, i32, i32, i32, vp, vp, vp]
        pp, i64s = C.c_void_p, C.c_int64
        L.obs_paged_init.argtypes = [vp, C.POINTER(PagedConfig)]
        L.obs_paged_append.argtypes = [vp, pp, vp, vp, i64s, vp, vp, i32, vp]
        L.obs_paged_decode.argtypes = [vp, pp, vp, i64s, vp, i32, i32, C.c_float, vp, i32, vp]
        L.obs_paged_prefill.argtypes = [vp, pp, vp, i64s, vp, vp, i32, i32, i32, C.c_float, vp]
        L.obs_paged_evict.argtypes = [vp, pp, pp, vp, vp, i32, i32, i32, i32, vp, vp, vp]
        L.obs_paged_attn_forward.argtypes = [vp, i32, pp, vp, vp, i32, vp, vp, vp, vp, i32, i32, vp, i32, vp]
        L.obs_paged_struct_layout.argtypes = [C.POINTER(C.c_int32), i32]
        L.obs_set_wait_limit.argtypes = [vp, i64]
        L.obs_probe_wait.argtypes = [vp, vp]
        L.obs_struct_layout.argtypes = [C.POINTER(C.c_int32), i32]
        L.obs_decode_ffn_static.argtypes = [C.POINTER(LayerWeights), i32, i32, i32, i32, vp, vp, vp, vp, i32, vp, vp]
        for name in EXPORTS:
            if name not in ("obs_last_error", "obs_abi_version"):
                getattr(L, name).restype = i32
        _LIB = L
    return _LIB


def _ptr(x) -> int | None:
    if x is None:
        return None
    if isinstance(x, int):
        return x
    if hasattr(x, "data_ptr"):
        return x.data_ptr()
    if hasattr(x, "ctypes"):  # numpy array (host memory)
        return x.ctypes.data
    raise TypeError(f"cannot take a pointer of {type(x)}")


def _stream(s) -> int | None:
    if s is None:
        return None
    if isinstance(s, int):
        return s
    return s.cuda_stream  # torch.cuda.Stream


@dataclass
class MoeShape:
    hidden: int = 2048
    inter: int = 768
    n_experts: int = 128
    top_k: int = 8
    n_layers: int = 1
    max_tokens: int = 512
    norm_topk: bool = True
    decode_max_tokens: int = 0   # <= 0: the library's default
    rms_eps: float = 1e-6
    ep_world: int = 1    # expert parallelism: ranks sharing the experts
    ep_rank: int = 0


class MoeContext:
    """One GPU's HBM-resident MoE layers (obs_create ... obs_destroy)."""

    def __init__(self, shape: MoeShape, device: int = 0):
        self.shape = shape
        cfg = Config(shape.hidden, shape.inter, shape.n_experts, shape.top_k, 64, shape.n_layers,
                     shape.max_tokens, int(shape.norm_topk), shape.decode_max_tokens, shape.rms_eps,
                     shape.ep_world, shape.ep_rank)
        h = C.c_void_p()
        rc = lib().obs_create(C.byref(cfg), device, C.byref(h))
        if rc != OBS_OK:
            raise ObsError(rc, lib().obs_last_error(None).decode())
        self._h = h
        self.device = device

    # -- plumbing
    def _chk(self, rc: int):
        if rc != OBS_OK:
            raise ObsError(rc, lib().obs_last_error(self._h).decode())

    def close(self):
        if getattr(self, "_h", None):
            lib().obs_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def memory_bytes(self):
        w, s = C.c_size_t(), C.c_size_t()
        self._chk(lib().obs_memory_bytes(self._h, C.byref(w), C.byref(s)))
        return w.value, s.value

    # -- weights
    def load_layer(self, layer: int, w, on_device: bool = False):
        """Copy one layer in the reference format (attributes router_w ... down_b)."""
        lw = LayerWeights(*[_ptr(getattr(w, n)) for n, _ in LayerWeights._fields_])
        self._chk(lib().obs_load_layer(self._h, layer, C.byref(lw), int(on_device)))

    def load_layer_file(self, layer: int, path: str, router_w, router_s, router_b):
        """One layer from the reference splitter's safetensors file (experts) plus the router
        arrays (host numpy arrays in the MLX layout)."""
        self._chk(lib().obs_load_layer_safetensors(self._h, layer, os.fsencode(path), _ptr(router_w), _ptr(router_s),
                                                   _ptr(router_b)))

    def load_head(self, vocab: int, w, on_device: bool = False):
        """The embedding, final norm and lm_head (attributes embed_w ... norm_w)."""
        hw = HeadWeights(*[_ptr(getattr(w, n)) for n, _ in HeadWeights._fields_])
        self._chk(lib().obs_load_head(self._h, vocab, C.byref(hw), int(on_device)))

    def embed(self, tokens, T, x, stream=None):
        self._chk(lib().obs_embed(self._h, _ptr(tokens), T, _ptr(x), _stream(stream)))

    def lm_head(self, x, T, ids, logits=None, stream=None):
        """RMSNorm(model.norm) -> lm_head -> greedy ids (first maximum); logits optional."""
        self._chk(lib().obs_lm_head(self._h, _ptr(x), T, _ptr(ids), _ptr(logits), _stream(stream)))

    # -- the attention block
    def attn_init(self, n_heads=32, n_kv_heads=4, head_dim=128, max_seq=4096, n_seqs=1, rope_theta=1e7):
        ac = AttnConfig(n_heads, n_kv_heads, head_dim, max_seq, n_seqs, rope_theta)
        self._chk(lib().obs_attn_init(self._h, C.byref(ac)))

    def load_attn(self, layer: int, w, on_device: bool = False):
        """One layer's attention weights (attributes q_w ... k_norm, MLX 4-bit layout)."""
        aw = AttnWeights(*[_ptr(getattr(w, n)) for n, _ in AttnWeights._fields_])
        self._chk(lib().obs_load_attn(self._h, layer, C.byref(aw), int(on_device)))

    def attn_forward(self, layer, x, out, T, seq, pos, stream=None):
        """out = x + attention(x) for T tokens of sequences seq[t] at positions pos[t]; appends K/V."""
        self._chk(lib().obs_attn_forward(self._h, layer, _ptr(x), _ptr(out), T, _ptr(seq), _ptr(pos),
                                         _stream(stream)))

    def kv_read(self, layer, seq, pos0, n, k=None, v=None, stream=None):
        self._chk(lib().obs_kv_read(self._h, layer, seq, pos0, n, _ptr(k), _ptr(v), _stream(stream)))

    # -- the paged key/value cache
    def paged_init(self, n_heads=32, n_kv_heads=4, head_dim=128, page_size=64, max_seqs=1, max_kv_len=4096,
                   dtype="bf16", weights=False):
        """The shape of the paged cache and its workspace (once per context); weights: decode steps
        may add up attention weights."""
        if dtype not in _DTYPES:
            raise ValueError(f"dtype must be one of {sorted(_DTYPES)}")
        pc = PagedConfig(n_heads, n_kv_heads, head_dim, page_size, max_seqs, max_kv_len, _DTYPES[dtype], int(weights))
        self._chk(lib().obs_paged_init(self._h, C.byref(pc)))
        plan = (page_size, n_kv_heads, head_dim, dtype)
        self._paged = _PLANS.setdefault(plan, plan)
        self._paged_row, self._paged_kv_row = n_heads * head_dim, n_kv_heads * head_dim

    _paged = None  # page_size, n_kv_heads, head_dim, dtype after paged_init
    _paged_kv_row = 0

    def _paged_kv(self, kv):
        if kv.plan is not self._paged and self._paged is not None:
            raise ValueError(f"the cache's pages are {kv.plan}, the context's {self._paged}")
        return kv.ref

    def _paged_q(self, kv, q, out, rows):
        """q's row stride, after checks of q and out ([rows, n_heads, head_dim] or [rows, n_heads * head_dim])."""
        if self._paged is None:  # (the library says what is missing)
            return 0
        row = self._paged_row
        if q.dtype is not kv.dtype or out.dtype is not kv.dtype or not q.is_cuda or not out.is_cuda:
            raise ValueError(f"q and out must hold {kv.dtype} like the cache, on the GPU")
        if q.numel() != rows * row or out.numel() != rows * row:
            raise ValueError(f"q and out must be [{rows}, {row}]")
        if not out.is_contiguous():
            raise ValueError("out must be consecutive")
        if q.is_contiguous():
            return row
        if q.shape[0] != rows or (rows and not q[0].is_contiguous()):
            raise ValueError("each row of q must be consecutive")
        return q.stride(0) if rows > 1 else row

    @staticmethod
    def _paged_i32(kv, name, t, least):
        """The address of `least` consecutive int32 on the GPU (an int is an address, None stays)."""
        if t is None or t.__class__ is int:
            return t
        if t.numel() < least or not t.is_contiguous() or not t.is_cuda \
                or (t.dtype is not kv.i32 and (t.element_size() != 4 or t.is_floating_point())):
            raise ValueError(f"{name}: {least} consecutive int32 on the GPU")
        return t.data_ptr()

    def _paged_w(self, kv, w):
        if w is None:
            return None, 0
        if w.dim() != 3 or w.shape[0] != kv.n_seqs or w.shape[1] != kv.kv_shape[1] or w.element_size() != 4 \
                or not w.is_floating_point() or not w.is_contiguous() or not w.is_cuda:
            raise ValueError("weights: consecutive fp32 [n_seqs, n_kv_heads, positions] on the GPU")
        return w.data_ptr(), w.shape[2]

    def paged_append(self, kv, k, v, seq, slot, T, stream=None):
        """Rows k, v [T, n_kv_heads, head_dim] to positions slot[t] of sequences seq[t]."""
        ref = self._paged_kv(kv)
        stride = row = self._paged_kv_row
        if k.dtype is not kv.dtype or v.dtype is not kv.dtype or k.numel() < T * row or v.numel() < T * row \
                or not k.is_cuda or not v.is_cuda:
            raise ValueError(f"k and v must be [T, {row}] of {kv.dtype} on the GPU")
        if not (k.is_contiguous() and v.is_contiguous()) and T:
            if k.shape[0] < T or v.shape[0] < T or not k[0].is_contiguous() or not v[0].is_contiguous() \
                    or (T > 1 and k.stride(0) != v.stride(0)):
                raise ValueError("each row of k and v must be consecutive, their strides the same")
            stride = k.stride(0) if T > 1 else row
        # (a decode step's append takes less time on the GPU than here: no calls that it can do without)
        rc = (_LIB or lib()).obs_paged_append(self._h, ref, k.data_ptr(), v.data_ptr(), stride,
                                              self._paged_i32(kv, "seq", seq, T), self._paged_i32(kv, "slot", slot, T), T,
                                              stream if stream is None else _stream(stream))
        if rc:
            self._chk(rc)

    def paged_decode(self, kv, q, out, window=0, n_sink=0, scale=0.0, weights=None, stream=None):
        """Attention of each sequence's last position over its pages; weights (optional) += the probabilities."""
        ref = self._paged_kv(kv)
        w, ws = self._paged_w(kv, weights)
        self._chk((_LIB or lib()).obs_paged_decode(self._h, ref, q.data_ptr(), self._paged_q(kv, q, out, kv.n_seqs),
                                                   out.data_ptr(), window, n_sink, scale, w, ws, _stream(stream)))

    def paged_prefill(self, kv, q, out, q_start, T, window=0, n_sink=0, scale=0.0, stream=None):
        """Attention of the sequences' last positions, rows q_start[s] .. q_start[s+1] of q each."""
        ref = self._paged_kv(kv)
        self._chk((_LIB or lib()).obs_paged_prefill(self._h, ref, q.data_ptr(), self._paged_q(kv, q, out, T),
                                                    out.data_ptr(), self._paged_i32(kv, "q_start", q_start, kv.n_seqs + 1),
                                                    T, window, n_sink, scale, _stream(stream)))

    def paged_evict(self, kv, dst, weights, weights_dst, budget, n_sink=0, n_recent=0, kept=None, new_len=None,
                    stream=None):
        """Keeps `budget` positions per sequence and KV head, moved to dst; kept int32 [n_seqs,
        n_kv_heads, budget] and new_len int32 [n_seqs] are written."""
        ref, to = self._paged_kv(kv), self._paged_kv(dst)
        w, ws = self._paged_w(kv, weights)
        wd, wds = self._paged_w(kv, weights_dst)
        if wd is not None and wds != ws:
            raise ValueError("weights and weights_dst must have one shape")
        self._chk(lib().obs_paged_evict(self._h, ref, to, w, wd, ws, budget, n_sink, n_recent,
                                        self._paged_i32(kv, "kept", kept, kv.n_seqs * kv.kv_shape[1] * budget),
                                        self._paged_i32(kv, "new_len", new_len, kv.n_seqs), _stream(stream)))

    def paged_attn_forward(self, layer, kv, x, out, T, seq, pos, slot, q_start=None, window=0, n_sink=0, weights=None,
                           stream=None):
        """attn_forward over a paged cache: a decode step (q_start None) or prompts' new tokens."""
        w, ws = self._paged_w(kv, weights)
        for t in (x, out):
            if t is not None and not isinstance(t, int) and (t.element_size() != 2 or t.numel() < T * self.shape.hidden
                                                             or not t.is_contiguous() or not t.is_cuda):
                raise ValueError(f"x and out must be consecutive bf16 [T, {self.shape.hidden}] on the GPU")
        self._chk(lib().obs_paged_attn_forward(self._h, layer, self._paged_kv(kv), _ptr(x), _ptr(out), T,
                                               self._paged_i32(kv, "seq", seq, T), self._paged_i32(kv, "pos", pos, T),
                                               self._paged_i32(kv, "slot", slot, T),
                                               self._paged_i32(kv, "q_start", q_start, kv.n_seqs + 1), window, n_sink, w, ws,
                                               _stream(stream)))

    def synth_layer(self, layer: int, seed: int = 0):
        self._chk(lib().obs_synth_layer(self._h, layer, seed))

    # -- the reference helpers
    def gate_gpu(self, layer, x, logits, T, stream=None):
        self._chk(lib().obs_gate(self._h, layer, _ptr(x), _ptr(logits), T, _stream(stream)))

    def route(self, logits, T, ids, weights, bias=None, stream=None):
        self._chk(lib().obs_route(self._h, _ptr(logits), _ptr(bias), T, _ptr(ids), _ptr(weights),
                                  _stream(stream)))

    def dispatch(self, ids, T, counts=None, seg=None, slot_of=None, stream=None):
        self._chk(lib().obs_dispatch(self._h, _ptr(ids), T, _ptr(counts), _ptr(seg), _ptr(slot_of),
                                     _stream(stream)))

    def expert_ffn(self, layer, x, ids, T, y, path=PATH_PREFILL, stream=None):
        self._chk(lib().obs_expert_ffn(self._h, layer, _ptr(x), _ptr(ids), T, path, _ptr(y),
                                       _stream(stream)))

    def matmul_raw_f32(self, layer, proj, expert, x, n, y, stream=None):
        """One expert projection on the tcgen05 GEMM, fp32 out (matmul_dequant_4bit)."""
        self._chk(lib().obs_expert_gemm_f32(self._h, layer, proj, expert, _ptr(x), n, _ptr(y),
                                            _stream(stream)))

    # -- expert parallelism
    def ep_handle(self) -> bytes:
        """This rank's buffer handle (obs_ep_handle), to be sent to the other ranks."""
        buf = (C.c_uint8 * EP_HANDLE_BYTES)()
        self._chk(lib().obs_ep_handle(self._h, buf))
        return bytes(buf)

    def ep_connect(self, handles):
        """Open every rank's buffer (obs_ep_connect); handles in rank order."""
        blob = b"".join(handles)
        assert len(blob) == EP_HANDLE_BYTES * self.shape.ep_world
        buf = (C.c_uint8 * len(blob)).from_buffer_copy(blob)
        self._chk(lib().obs_ep_connect(self._h, buf))

    def ep_set_placement(self, layer, experts):
        """Which GPU holds which expert (obs_ep_set_placement): experts[g*E/G + l] is GPU g's local
        expert l; layer = -1 for every layer.  Changed layers must be loaded again."""
        arr = (C.c_int32 * self.shape.n_experts)(*[int(e) for e in experts])
        self._chk(lib().obs_ep_set_placement(self._h, layer, arr))

    def ep_get_placement(self, layer) -> list:
        arr = (C.c_int32 * self.shape.n_experts)()
        self._chk(lib().obs_ep_get_placement(self._h, layer, arr))
        return list(arr)

    def moe_forward(self, layer, x, out, T, residual=None, bias=None, path=PATH_AUTO, stream=None):
        self._chk(lib().obs_moe_forward(self._h, layer, _ptr(x), _ptr(out), _ptr(residual), T,
                                        _ptr(bias), path, _stream(stream)))

    def rmsnorm(self, x, out, T, weight=None, stream=None):
        self._chk(lib().obs_rmsnorm(self._h, _ptr(x), _ptr(weight), T, _ptr(out), _stream(stream)))

    def moe_stack_forward(self, layer0, n_layers, resid, T, bias=None, path=PATH_AUTO, stream=None):
        """resid <- n_layers of (r + MoE_l(RMSNorm(r))), in place."""
        self._chk(lib().obs_moe_stack_forward(self._h, layer0, n_layers, _ptr(resid), T, _ptr(bias), path,
                                              _stream(stream)))

    def moe_forward_host(self, layer, x_host, out_host, T, residual_host=None, bias_host=None,
                         path=PATH_AUTO, stream=None):
        self._chk(lib().obs_moe_forward_host(self._h, layer, _ptr(x_host), _ptr(out_host),
                                             _ptr(residual_host), T, _ptr(bias_host), path,
                                             _stream(stream)))

    def moe_forward_host_async(self, layer, x_host, out_host, T, residual_host=None, bias_host=None,
                               path=PATH_AUTO, stream=None):
        """moe_forward_host without the wait: copies in and out on internal streams, two staging
        slots, so successive calls overlap (host_join, then synchronise, before reading out_host)."""
        self._chk(lib().obs_moe_forward_host_async(self._h, layer, _ptr(x_host), _ptr(out_host),
                                                   _ptr(residual_host), T, _ptr(bias_host), path,
                                                   _stream(stream)))

    def host_join(self, stream=None):
        """Make `stream` wait for every output copy moe_forward_host_async has issued."""
        self._chk(lib().obs_moe_host_join(self._h, _stream(stream)))

    def profile(self, enable: bool):
        self._chk(lib().obs_profile_enable(self._h, int(enable)))

    def profile_read(self) -> dict:
        """{stage: (total ms, launches)} since the last read (event times on the caller's stream)."""
        ms = (C.c_float * len(STAGES))()
        n = (C.c_int32 * len(STAGES))()
        self._chk(lib().obs_profile_read(self._h, ms, n))
        return {name: (ms[i], n[i]) for i, name in enumerate(STAGES)}

    def trace(self, buf, n_steps: int):
        """Record the gate/up GEMM pipeline timeline of CTA 0 into buf (uint64 [8, n_steps])."""
        self._chk(lib().obs_trace_enable(self._h, _ptr(buf), n_steps if buf is not None else 0))

    def debug_gemm_tiles(self, layer, tiles, stream=None):
        """Test hook: the gate/up GEMM over a given tile list (numpy int32 [n][4])."""
        import numpy as np

        t = np.ascontiguousarray(tiles, dtype=np.int32).reshape(-1, 4)
        self._chk(lib().obs_debug_gemm_tiles(self._h, layer, t.ctypes.data, len(t), _stream(stream)))

    def check_device(self, stream=None):
        self._chk(lib().obs_check_device(self._h, _stream(stream)))

    def set_wait_limit(self, limit_ns: int):
        """Limit of every bounded device-side wait (0: the default 2 s)."""
        self._chk(lib().obs_set_wait_limit(self._h, limit_ns))

    def probe_wait(self, stream=None):
        """One bounded device wait on a stamp nothing writes: it runs out after the wait limit."""
        self._chk(lib().obs_probe_wait(self._h, _stream(stream)))


def decode_ffn_static(w, n_experts, hidden, inter, top_k, x, ids, weights, T, out, residual=None, stream=None):
    """obs_decode_ffn_static: the decode FFN + combine with no context and no
    device allocation (scratch is a fixed array inside the library).  ``w``
    holds device buffers of the expert weights in the reference (MLX) layout."""
    lw = LayerWeights(None, None, None, *[_ptr(getattr(w, n)) for n, _ in LayerWeights._fields_[3:]])
    rc = lib().obs_decode_ffn_static(C.byref(lw), n_experts, hidden, inter, top_k, _ptr(x), _ptr(ids),
                                     _ptr(weights), _ptr(residual), T, _ptr(out), _stream(stream))
    if rc != OBS_OK:
        raise ObsError(rc, lib().obs_last_error(None).decode())


def expert_file_info(path: str) -> tuple[int, int, int]:
    """(n_experts, hidden, inter) of a splitter expert file, read from its header alone."""
    e, h, i = C.c_int32(), C.c_int32(), C.c_int32()
    rc = lib().obs_expert_file_info(os.fsencode(path), C.byref(e), C.byref(h), C.byref(i))
    if rc != OBS_OK:
        raise ObsError(rc, lib().obs_last_error(None).decode())
    return e.value, h.value, i.value


def plan_placement(load, world: int) -> list:
    """A balanced expert placement from per-expert loads (obs_ep_plan_placement; host only)."""
    E = len(load)
    lo = (C.c_int64 * E)(*[int(v) for v in load])
    out = (C.c_int32 * E)()
    rc = lib().obs_ep_plan_placement(lo, E, world, out)
    if rc != 0:
        raise ObsError(rc, "obs_ep_plan_placement: bad arguments")
    return list(out)


def paged_struct_layout() -> list[int]:
    """sizeof and field offsets of obs_paged_config and obs_paged_kv, as the library was compiled."""
    n = lib().obs_paged_struct_layout(None, 0)
    buf = (C.c_int32 * n)()
    lib().obs_paged_struct_layout(buf, n)
    return list(buf)


def struct_layout() -> list[int]:
    """sizeof and field offsets of obs_config and obs_layer_weights, as the library was compiled."""
    n = lib().obs_struct_layout(None, 0)
    buf = (C.c_int32 * n)()
    lib().obs_struct_layout(buf, n)
    return list(buf)


def kernel_launches() -> int:
    """Kernel launches the library has issued in this process (all contexts)."""
    n = C.c_uint64(0)
    rc = lib().obs_kernel_launches(C.byref(n))
    if rc != OBS_OK:
        raise ObsError(rc, "kernel_launches")
    return int(n.value)


def synth_activations(seed, layer, row0, T, H, x, eps=1e-6, stream=None):
    rc = lib().obs_synth_activations(seed, layer, row0, T, H, eps, _ptr(x), _stream(stream))
    if rc != OBS_OK:
        raise ObsError(rc, "synth_activations")
