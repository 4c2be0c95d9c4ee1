"""ctypes binding of libkatago_cuda.so.

Mirrors the reference backend's NeuralNet steps (crates/katago-nn-burn/src/backend.rs): Model.load ~
load_model_file, Context ~ create_compute_context, Handle ~ create_compute_handle + create_input_buffers,
Handle.get_output ~ get_output, and the asynchronous halves Handle.enqueue / Handle.wait of run_network.
"""

from __future__ import annotations

import ctypes
import os
import struct
from typing import Optional, Sequence

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.dirname(os.path.dirname(HERE))  # katago-rs_b200/
HEADER = os.path.join(os.path.dirname(PKG), "include", "katago_cuda.h")

PRECISION_F32, PRECISION_F16, PRECISION_BF16, PRECISION_AUTO = 0, 1, 2, 3
ACT_IDENTITY, ACT_RELU, ACT_MISH, ACT_SILU = range(4)
ROPE_HALVES, ROPE_PAIRS = 0, 1
ROPE_MAX_AXES = 4
NORM_LAYER, NORM_RMS = 0, 1
KC_OK, KC_ERR_INVALID, KC_ERR_PARSE, KC_ERR_CUDA, KC_ERR_TIMEOUT, KC_ERR_DEVICE, KC_ERR_NO_DEVICE = range(7)

_LIB = None


def library_path() -> str:
    return os.environ.get("KATAGO_CUDA_LIB", os.path.join(PKG, "lib", "libkatago_cuda.so"))


class KcError(RuntimeError):
    def __init__(self, status: int, msg: str):
        super().__init__(msg)
        self.status = status


class Desc(ctypes.Structure):
    _fields_ = [
        ("name", ctypes.c_char * 128),
        ("model_version", ctypes.c_int32),
        ("num_input_channels", ctypes.c_int32),
        ("num_input_global_channels", ctypes.c_int32),
        ("num_input_meta_channels", ctypes.c_int32),
        ("meta_encoder_version", ctypes.c_int32),
        ("num_policy_channels", ctypes.c_int32),
        ("num_value_channels", ctypes.c_int32),
        ("num_score_value_channels", ctypes.c_int32),
        ("num_ownership_channels", ctypes.c_int32),
        ("trunk_num_blocks", ctypes.c_int32),
        ("trunk_num_channels", ctypes.c_int32),
        ("trunk_norm_kind", ctypes.c_int32),
        ("has_any_transformer_blocks", ctypes.c_int32),
        ("has_any_nested_bottleneck_blocks", ctypes.c_int32),
        ("post_process_from_header", ctypes.c_int32),
        ("prefer_pass_alive_under_suicide_rules", ctypes.c_int32),
        ("prefer_exclude_territory_adjacent_to_atari", ctypes.c_int32),
        ("num_parameters", ctypes.c_int64),
        ("trunk_spatial_conv_depth", ctypes.c_double),
        ("post_process", ctypes.c_float * 8),
    ]


class GroupNormDesc(ctypes.Structure):
    """kc_group_norm_desc. dtype: PRECISION_*, act: ACT_*; x_strides, y_strides: (board, row) strides in elements,
    None = contiguous; mask_stride: elements from one board's mask to the next, None = points."""

    _fields_ = [
        ("dtype", ctypes.c_int32),
        ("act", ctypes.c_int32),
        ("n", ctypes.c_int32),
        ("points", ctypes.c_int32),
        ("channels", ctypes.c_int32),
        ("groups", ctypes.c_int32),
        ("eps", ctypes.c_float),
        ("reserved", ctypes.c_int32),
        ("x_board_stride", ctypes.c_int64),
        ("x_row_stride", ctypes.c_int64),
        ("y_board_stride", ctypes.c_int64),
        ("y_row_stride", ctypes.c_int64),
        ("mask_board_stride", ctypes.c_int64),
    ]

    def __init__(self, dtype, act, n, points, channels, groups, eps, x_strides=None, y_strides=None,
                 mask_stride=None):
        whole = (points * channels, channels)
        self._pack(self, 0, dtype, act, n, points, channels, groups, eps, 0, *(x_strides or whole),
                   *(y_strides or whole), points if mask_stride is None else mask_stride)

    _pack = struct.Struct("=6ifi5q").pack_into  # the fields in one go: made for every call of small batches


class LayerNormDesc(ctypes.Structure):
    """kc_layer_norm_desc. dtype: PRECISION_*, kind: NORM_*; strides as GroupNormDesc's."""

    _fields_ = [
        ("dtype", ctypes.c_int32),
        ("kind", ctypes.c_int32),
        ("n", ctypes.c_int32),
        ("points", ctypes.c_int32),
        ("channels", ctypes.c_int32),
        ("eps", ctypes.c_float),
        ("x_board_stride", ctypes.c_int64),
        ("x_row_stride", ctypes.c_int64),
        ("y_board_stride", ctypes.c_int64),
        ("y_row_stride", ctypes.c_int64),
        ("mask_board_stride", ctypes.c_int64),
    ]

    def __init__(self, dtype, kind, n, points, channels, eps, x_strides=None, y_strides=None, mask_stride=None):
        whole = (points * channels, channels)
        self._pack(self, 0, dtype, kind, n, points, channels, eps, *(x_strides or whole), *(y_strides or whole),
                   points if mask_stride is None else mask_stride)

    _pack = struct.Struct("=5if5q").pack_into


class EmbedDesc(ctypes.Structure):
    """kc_embed_desc. dtype: PRECISION_*; strides in elements, None = contiguous rows."""

    _fields_ = [
        ("dtype", ctypes.c_int32),
        ("channels", ctypes.c_int32),
        ("tokens", ctypes.c_int64),
        ("table_rows", ctypes.c_int64),
        ("scale", ctypes.c_float),
        ("reserved", ctypes.c_int32),
        ("table_stride", ctypes.c_int64),
        ("x_stride", ctypes.c_int64),
        ("y_stride", ctypes.c_int64),
    ]

    def __init__(self, dtype, tokens, channels, table_rows, scale=1.0, table_stride=None, x_stride=None,
                 y_stride=None):
        strides = (channels if s is None else s for s in (table_stride, x_stride, y_stride))
        self._pack(self, 0, dtype, channels, tokens, table_rows, scale, 0, *strides)

    _pack = struct.Struct("=2i2qfi3q").pack_into


class DistillDesc(ctypes.Structure):
    """kc_distill_desc. dtype: PRECISION_*; strides in elements, None = contiguous rows."""

    _fields_ = [
        ("dtype", ctypes.c_int32),
        ("classes", ctypes.c_int32),
        ("rows", ctypes.c_int64),
        ("top", ctypes.c_int32),
        ("temperature", ctypes.c_float),
        ("logits_stride", ctypes.c_int64),
        ("dlogits_stride", ctypes.c_int64),
        ("top_stride", ctypes.c_int64),
    ]

    def __init__(self, dtype, rows, classes, top, temperature=1.0, logits_stride=None, dlogits_stride=None,
                 top_stride=None):
        self._pack(self, 0, dtype, classes, rows, top, temperature, classes if logits_stride is None else logits_stride,
                   classes if dlogits_stride is None else dlogits_stride, top if top_stride is None else top_stride)

    _pack = struct.Struct("=2iqif3q").pack_into


class RopeDesc(ctypes.Structure):
    """kc_rope_desc. dtype: PRECISION_*, layout: ROPE_*; the strides are (token, head) in elements, None =
    contiguous [tokens][heads][head_dim]."""

    _fields_ = [
        ("dtype", ctypes.c_int32),
        ("layout", ctypes.c_int32),
        ("axes", ctypes.c_int32),
        ("q_heads", ctypes.c_int32),
        ("k_heads", ctypes.c_int32),
        ("head_dim", ctypes.c_int32),
        ("rotary_dim", ctypes.c_int32),
        ("tables", ctypes.c_int32),
        ("tokens", ctypes.c_int64),
        ("q_token_stride", ctypes.c_int64),
        ("q_head_stride", ctypes.c_int64),
        ("k_token_stride", ctypes.c_int64),
        ("k_head_stride", ctypes.c_int64),
        ("q_out_token_stride", ctypes.c_int64),
        ("q_out_head_stride", ctypes.c_int64),
        ("k_out_token_stride", ctypes.c_int64),
        ("k_out_head_stride", ctypes.c_int64),
    ]

    def __init__(self, dtype, layout, axes, tokens, q_heads, k_heads, head_dim, rotary_dim, tables=1, q_strides=None,
                 k_strides=None, q_out_strides=None, k_out_strides=None):
        q, k = (q_heads * head_dim, head_dim), (k_heads * head_dim, head_dim)
        self._pack(self, 0, dtype, layout, axes, q_heads, k_heads, head_dim, rotary_dim, tables, tokens,
                   *(q_strides or q), *(k_strides or k), *(q_out_strides or q), *(k_out_strides or k))

    _pack = struct.Struct("=8i9q").pack_into


P = ctypes.c_void_p
I = ctypes.c_int
FP = ctypes.POINTER(ctypes.c_float)
FPP = ctypes.POINTER(FP)

_SIGS = {
    "kc_last_error": ([], ctypes.c_char_p),
    "kc_device_count": ([ctypes.POINTER(I)], I),
    "kc_model_load": ([ctypes.c_char_p, ctypes.c_size_t, ctypes.c_char_p, ctypes.POINTER(P)], I),
    "kc_model_desc": ([P, ctypes.POINTER(Desc)], I),
    "kc_model_destroy": ([P], I),
    "kc_model_flops": ([P, ctypes.POINTER(ctypes.c_double), ctypes.POINTER(ctypes.c_double)], I),
    "kc_context_create": ([ctypes.POINTER(I), I, I, I, I, P, ctypes.POINTER(P)], I),
    "kc_context_precision": ([P, ctypes.POINTER(I)], I),
    "kc_context_destroy": ([P], I),
    "kc_handle_create": ([P, I, I, I, ctypes.POINTER(P)], I),
    "kc_handle_destroy": ([P], I),
    "kc_handle_input_ptrs": ([P, FPP, FPP, FPP], I),
    "kc_handle_output_layout": ([P] + [ctypes.POINTER(I)] * 5, I),
    "kc_enqueue": ([P, I], I),
    "kc_wait": ([P, I, FPP], I),
    "kc_enqueue_device": ([P, I, P, P, P, P], I),
    "kc_synchronize": ([P, I], I),
    "kc_handle_stream": ([P, ctypes.POINTER(P)], I),
    "kc_get_output": ([P, I, FPP, FPP, FPP, ctypes.POINTER(I), FP, I, FP, FP, FP, FP], I),
    "kc_handle_set_profiling": ([P, I], I),
    "kc_handle_profile": ([P, ctypes.POINTER(ctypes.c_double), ctypes.POINTER(ctypes.c_int64), I], I),
    "kc_handle_launch_count": ([P, I, ctypes.POINTER(I)], I),
    "kc_copy_with_symmetry": ([FP, FP, I, I, I, I, I, I], I),
    "kc_gpool_fc": ([P, P, I, I, P, I, P, P], I),
    "kc_gpool_fc_noalloc": ([P, P, I, I, P, I, P, P], I),
    "kc_group_norm_act_workspace": ([ctypes.POINTER(GroupNormDesc), I, ctypes.POINTER(ctypes.c_size_t)], I),
    "kc_group_norm_act": ([ctypes.POINTER(GroupNormDesc), P, P, P, P, P, P, P, ctypes.c_size_t, P], I),
    "kc_group_norm_act_backward": ([ctypes.POINTER(GroupNormDesc)] + [P] * 10 + [ctypes.c_size_t, P], I),
    "kc_rope_axes_freqs": ([I, ctypes.POINTER(ctypes.c_int32), ctypes.c_double, I, FP], I),
    "kc_rope_axes": ([ctypes.POINTER(RopeDesc), P, P, P, P, P, P, P], I),
    "kc_rope_axes_backward_workspace": ([ctypes.POINTER(RopeDesc), ctypes.POINTER(ctypes.c_size_t)], I),
    "kc_rope_axes_backward": ([ctypes.POINTER(RopeDesc)] + [P] * 10 + [ctypes.c_size_t, P], I),
    "kc_layer_norm": ([ctypes.POINTER(LayerNormDesc)] + [P] * 7, I),
    "kc_layer_norm_backward_workspace": ([ctypes.POINTER(LayerNormDesc), ctypes.POINTER(ctypes.c_size_t)], I),
    "kc_layer_norm_backward": ([ctypes.POINTER(LayerNormDesc)] + [P] * 9 + [ctypes.c_size_t, P], I),
    "kc_embed_rows": ([ctypes.POINTER(EmbedDesc)] + [P] * 5, I),
    "kc_embed_rows_backward_workspace": ([ctypes.POINTER(EmbedDesc), ctypes.POINTER(ctypes.c_size_t)], I),
    "kc_embed_rows_backward": ([ctypes.POINTER(EmbedDesc)] + [P] * 4 + [ctypes.c_size_t, P], I),
    "kc_distill_top": ([ctypes.POINTER(DistillDesc)] + [P] * 7, I),
    "kc_distill_top_backward": ([ctypes.POINTER(DistillDesc)] + [P] * 8, I),
    "kc_selftest_device_timeout": ([P, I], I),
    "kc_handle_packed_input_ptrs": ([P, ctypes.POINTER(ctypes.POINTER(ctypes.c_uint32)), FPP, FPP,
                                     ctypes.POINTER(ctypes.POINTER(ctypes.c_int32)), FPP], I),
    "kc_enqueue_packed": ([P, I, I], I),
    "kc_pack_spatial": ([FP, I, ctypes.POINTER(ctypes.c_uint32)], I),
    "kc_symmetry_table": ([I, I, ctypes.POINTER(I)], I),
}
PACKED_WORDS_PER_PLANE = 12
FINISHED_ROW_LEN, FINISHED_POLICY, FINISHED_VALUE, FINISHED_MISC, FINISHED_OWNERSHIP = 732, 0, 362, 365, 371
GPOOL_NOALLOC_MAX_FLOATS = 262144


def lib():
    """The loaded library. Raises if it was not built (no fallback)."""
    global _LIB
    if _LIB is None:
        path = library_path()
        if not os.path.exists(path):
            raise RuntimeError(f"libkatago_cuda.so not found at {path}: build it with `make -C katago-rs_b200` "
                               f"(or __graft_entry__.build())")
        L = ctypes.CDLL(path)
        for name, (args, res) in _SIGS.items():
            f = getattr(L, name)
            f.argtypes = args
            f.restype = res
        _LIB = L
    return _LIB


def _check(rc: int):
    if rc != KC_OK:
        raise KcError(rc, lib().kc_last_error().decode(errors="replace"))


def _fp(a: np.ndarray):
    return a.ctypes.data_as(FP)


def device_count() -> int:
    c = I(0)
    _check(lib().kc_device_count(ctypes.byref(c)))
    return c.value


class Model:
    """A parsed model file (NeuralNet::load_model_file). No device is used."""

    def __init__(self, data: bytes, file_name: Optional[str] = "model.bin"):
        h = P()
        _check(lib().kc_model_load(data, len(data), file_name.encode() if file_name else None, ctypes.byref(h)))
        self.h = h
        d = Desc()
        _check(lib().kc_model_desc(self.h, ctypes.byref(d)))
        self.desc = d

    def flops(self):
        t, c3 = ctypes.c_double(), ctypes.c_double()
        _check(lib().kc_model_flops(self.h, ctypes.byref(t), ctypes.byref(c3)))
        return t.value, c3.value

    def close(self):
        if getattr(self, "h", None):
            lib().kc_model_destroy(self.h)
            self.h = None

    def __del__(self):
        self.close()


class Context:
    """NeuralNet::create_compute_context."""

    def __init__(self, model: Model, gpu_idxs: Sequence[int] = (-1,), precision: int = PRECISION_AUTO,
                 nn_x_len: int = 19, nn_y_len: int = 19):
        arr = (I * len(gpu_idxs))(*gpu_idxs)
        h = P()
        _check(lib().kc_context_create(arr, len(gpu_idxs), nn_x_len, nn_y_len, precision, model.h, ctypes.byref(h)))
        self.h = h
        self.model = model
        p = I()
        _check(lib().kc_context_precision(self.h, ctypes.byref(p)))
        self.precision = p.value

    def close(self):
        if getattr(self, "h", None):
            lib().kc_context_destroy(self.h)
            self.h = None

    def __del__(self):
        self.close()


class Handle:
    """NeuralNet::create_compute_handle plus its pinned input buffers."""

    def __init__(self, ctx: Context, max_batch: int, gpu_idx: int = -1):
        h = P()
        _check(lib().kc_handle_create(ctx.h, gpu_idx, max_batch, 0, ctypes.byref(h)))
        self.h = h
        self.ctx = ctx
        self.max_batch = max_batch
        d = ctx.model.desc
        self.n_spatial = d.num_input_channels * 361
        self.n_global = d.num_input_global_channels
        self.n_meta = d.num_input_meta_channels
        s, g, m = FP(), FP(), FP()
        _check(lib().kc_handle_input_ptrs(self.h, ctypes.byref(s), ctypes.byref(g), ctypes.byref(m)))
        self.spatial = np.ctypeslib.as_array(s, shape=(max_batch, d.num_input_channels, 19, 19))
        self.glob = np.ctypeslib.as_array(g, shape=(max_batch, self.n_global))
        self.meta = np.ctypeslib.as_array(m, shape=(max_batch, self.n_meta)) if self.n_meta else None
        vals = [I() for _ in range(5)]
        _check(lib().kc_handle_output_layout(self.h, *[ctypes.byref(v) for v in vals]))
        self.row_len, self.policy_off, self.value_off, self.score_off, self.own_off = [v.value for v in vals]
        self.P = d.num_policy_channels
        b, g, m, sy, op = (ctypes.POINTER(ctypes.c_uint32)(), FP(), FP(), ctypes.POINTER(ctypes.c_int32)(), FP())
        _check(lib().kc_handle_packed_input_ptrs(self.h, ctypes.byref(b), ctypes.byref(g), ctypes.byref(m),
                                                 ctypes.byref(sy), ctypes.byref(op)))
        self.pk_bits = np.ctypeslib.as_array(b, shape=(max_batch, d.num_input_channels, PACKED_WORDS_PER_PLANE))
        self.pk_glob = np.ctypeslib.as_array(g, shape=(max_batch, self.n_global))
        self.pk_meta = np.ctypeslib.as_array(m, shape=(max_batch, self.n_meta)) if self.n_meta else None
        self.pk_sym = np.ctypeslib.as_array(sy, shape=(max_batch,))
        self.pk_opt = np.ctypeslib.as_array(op, shape=(max_batch,))

    def close(self):
        if getattr(self, "h", None):
            lib().kc_handle_destroy(self.h)
            self.h = None

    def __del__(self):
        self.close()

    # ---- raw forward --------------------------------------------------------------------------------------------
    def enqueue(self, n: int):
        _check(lib().kc_enqueue(self.h, n))

    def wait(self, timeout_ms: int = -1) -> np.ndarray:
        """The n output rows of the last enqueue (a view of pinned memory, valid until the next enqueue)."""
        p = FP()
        _check(lib().kc_wait(self.h, timeout_ms, ctypes.byref(p)))
        return np.ctypeslib.as_array(p, shape=(self.max_batch, self.row_len))

    def forward(self, spatial, glob, meta=None, timeout_ms: int = 120000) -> dict:
        """Raw outputs of the reference graph for n rows: policy [n,P,362], value [n,3], scorevalue [n,Sv],
        ownership [n,1,19,19]."""
        n = spatial.shape[0]
        self.spatial[:n] = spatial
        self.glob[:n] = glob
        if self.n_meta:
            self.meta[:n] = meta
        self.enqueue(n)
        rows = np.array(self.wait(timeout_ms)[:n])
        return self.split(rows)

    def split(self, rows: np.ndarray) -> dict:
        n = rows.shape[0]
        return {
            "policy": rows[:, self.policy_off:self.policy_off + self.P * 362].reshape(n, self.P, 362),
            "value": rows[:, self.value_off:self.value_off + 3],
            "scorevalue": rows[:, self.score_off:self.own_off],
            "ownership": rows[:, self.own_off:self.own_off + 361].reshape(n, 1, 19, 19),
        }

    def enqueue_packed(self, n: int, finish: bool):
        """kc_enqueue_packed: rows [0, n) of the packed staging (pk_bits, pk_glob, pk_meta, pk_sym, pk_opt)."""
        _check(lib().kc_enqueue_packed(self.h, n, int(finish)))

    def wait_finished(self, timeout_ms: int = -1) -> np.ndarray:
        """The NNOutput rows [max_batch, FINISHED_ROW_LEN] of the last kc_enqueue_packed(finish=1)."""
        p = FP()
        _check(lib().kc_wait(self.h, timeout_ms, ctypes.byref(p)))
        return np.ctypeslib.as_array(p, shape=(self.max_batch, FINISHED_ROW_LEN))

    def forward_packed(self, spatial, glob, symmetry, meta=None, timeout_ms: int = 120000) -> dict:
        """Raw outputs (as forward) of n rows sent bit-packed with per-row symmetries applied on the device."""
        n = spatial.shape[0]
        for i in range(n):
            self.pk_bits[i] = pack_spatial(spatial[i])
        self.pk_glob[:n] = glob
        if self.n_meta:
            self.pk_meta[:n] = meta
        self.pk_sym[:n] = symmetry
        self.enqueue_packed(n, False)
        rows = np.array(self.wait(timeout_ms)[:n])
        return self.split(rows)

    def enqueue_device(self, n: int, d_spatial: int, d_global: int, d_meta: int, d_out: int):
        _check(lib().kc_enqueue_device(self.h, n, d_spatial, d_global, d_meta or None, d_out))

    def stream_ptr(self) -> int:
        s = P()
        _check(lib().kc_handle_stream(self.h, ctypes.byref(s)))
        return s.value or 0

    def synchronize(self, timeout_ms: int = -1):
        _check(lib().kc_synchronize(self.h, timeout_ms))

    def selftest_device_timeout(self, limit_us: int):
        """kc_selftest_device_timeout: enqueue a kernel whose bounded wait runs out after `limit_us`."""
        _check(lib().kc_selftest_device_timeout(self.h, limit_us))

    # ---- NeuralNet::get_output --------------------------------------------------------------------------------
    def get_output(self, spatial_rows, global_rows, meta_rows, symmetry, policy_optimism, want_ownership=True,
                   timeout_ms: int = 120000) -> dict:
        n = len(spatial_rows)
        sp = [np.ascontiguousarray(r, np.float32) for r in spatial_rows]
        gl = [np.ascontiguousarray(r, np.float32) for r in global_rows]
        sp_arr = (FP * n)(*[_fp(r) for r in sp])
        gl_arr = (FP * n)(*[_fp(r) for r in gl])
        me_arr = None
        if self.n_meta:
            me = [np.ascontiguousarray(r, np.float32) for r in meta_rows]
            me_arr = (FP * n)(*[_fp(r) for r in me])
        sym = (I * n)(*[int(s) for s in symmetry])
        opt = np.ascontiguousarray(policy_optimism, np.float32)
        pol = np.zeros((n, 362), np.float32)
        val = np.zeros((n, 3), np.float32)
        misc = np.zeros((n, 6), np.float32)
        own = np.zeros((n, 361), np.float32) if want_ownership else None
        _check(lib().kc_get_output(self.h, n, sp_arr, gl_arr, me_arr, sym, _fp(opt), timeout_ms, _fp(pol), _fp(val),
                                   _fp(misc), _fp(own) if own is not None else None))
        return {"policy": pol, "value": val, "misc": misc, "ownership": own}

    # ---- measurement ------------------------------------------------------------------------------------------
    def set_profiling(self, on: bool):
        _check(lib().kc_handle_set_profiling(self.h, int(on)))

    def profile(self):
        ms = (ctypes.c_double * 5)()
        n = (ctypes.c_int64 * 5)()
        _check(lib().kc_handle_profile(self.h, ms, n, 5))
        names = ["conv3x3", "linear", "stem", "attention", "other"]
        return {k: (ms[i], n[i]) for i, k in enumerate(names)}

    def launch_count(self, n: int) -> int:
        c = I()
        _check(lib().kc_handle_launch_count(self.h, n, ctypes.byref(c)))
        return c.value


def gpool_fc(d_x: int, d_mask: int, n: int, c: int, d_w: int, oc: int, d_out: int, stream: int = 0):
    """kc_gpool_fc on device pointers (masked global pooling + gpool-to-bias matmul)."""
    _check(lib().kc_gpool_fc(d_x, d_mask, n, c, d_w, oc, d_out, stream or None))


def gpool_fc_noalloc(d_x: int, d_mask: int, n: int, c: int, d_w: int, oc: int, d_out: int, stream: int = 0):
    """kc_gpool_fc_noalloc: the same operator with its scratch in a fixed device array (no allocation)."""
    _check(lib().kc_gpool_fc_noalloc(d_x, d_mask, n, c, d_w, oc, d_out, stream or None))


def group_norm_act_workspace(desc: GroupNormDesc, backward: bool) -> int:
    """kc_group_norm_act_workspace: bytes of device workspace a forward or backward call needs."""
    n = ctypes.c_size_t()
    _check(lib().kc_group_norm_act_workspace(desc, backward, n))
    return n.value


def group_norm_act(desc: GroupNormDesc, d_x: int, d_mask: int, d_weight: int, d_bias: int, d_y: int, d_stats: int = 0,
                   d_workspace: int = 0, workspace_bytes: int = 0, stream: int = 0):
    """kc_group_norm_act on device pointers (masked group norm and activation, channels last; 0 = not given)."""
    _check(lib().kc_group_norm_act(desc, d_x, d_mask, d_weight, d_bias, d_y, d_stats, d_workspace, workspace_bytes,
                                   stream))


def group_norm_act_backward(desc: GroupNormDesc, d_x: int, d_mask: int, d_weight: int, d_bias: int, d_stats: int,
                            d_dy: int, d_dx: int, d_dweight: int = 0, d_dbias: int = 0, d_workspace: int = 0,
                            workspace_bytes: int = 0, stream: int = 0):
    """kc_group_norm_act_backward on device pointers: the gradients by x, weight and bias."""
    _check(lib().kc_group_norm_act_backward(desc, d_x, d_mask, d_weight, d_bias, d_stats, d_dy, d_dx, d_dweight,
                                            d_dbias, d_workspace, workspace_bytes, stream))


def rope_axes_freqs(sections: Sequence[int], theta: float, rotary_dim: int) -> np.ndarray:
    """kc_rope_axes_freqs: fixed rotary frequencies [rotary_dim / 2, axes] float32, axis a turning sections[a] pairs."""
    axes = len(sections)
    out = np.zeros((max(0, rotary_dim // 2), axes), np.float32)
    _check(lib().kc_rope_axes_freqs(axes, (ctypes.c_int32 * axes)(*sections), theta, rotary_dim, _fp(out)))
    return out


def rope_axes(desc: RopeDesc, d_q: int, d_k: int, d_pos: int, d_freqs: int, d_q_out: int, d_k_out: int,
              stream: int = 0):
    """kc_rope_axes on device pointers: Q and K heads turned by their positions on several axes."""
    _check(lib().kc_rope_axes(desc, d_q, d_k, d_pos, d_freqs, d_q_out, d_k_out, stream))


def rope_axes_backward_workspace(desc: RopeDesc) -> int:
    """kc_rope_axes_backward_workspace: bytes of device workspace a backward call with d_dfreqs needs."""
    n = ctypes.c_size_t()
    _check(lib().kc_rope_axes_backward_workspace(desc, n))
    return n.value


def rope_axes_backward(desc: RopeDesc, d_dq_out: int, d_dk_out: int, d_q: int, d_k: int, d_pos: int, d_freqs: int,
                       d_dq: int, d_dk: int, d_dfreqs: int = 0, d_workspace: int = 0, workspace_bytes: int = 0,
                       stream: int = 0):
    """kc_rope_axes_backward on device pointers: the gradients by q, k and (d_dfreqs) the frequencies."""
    _check(lib().kc_rope_axes_backward(desc, d_dq_out, d_dk_out, d_q, d_k, d_pos, d_freqs, d_dq, d_dk, d_dfreqs,
                                       d_workspace, workspace_bytes, stream))


def layer_norm(desc: LayerNormDesc, d_x: int, d_mask: int, d_weight: int, d_bias: int, d_y: int, d_stats: int = 0,
               stream: int = 0):
    """kc_layer_norm on device pointers (layer or RMS norm of each token's row; 0 = not given)."""
    _check(lib().kc_layer_norm(desc, d_x, d_mask, d_weight, d_bias, d_y, d_stats, stream))


def layer_norm_backward_workspace(desc: LayerNormDesc) -> int:
    """kc_layer_norm_backward_workspace: bytes of device workspace a backward call with parameter gradients needs."""
    n = ctypes.c_size_t()
    _check(lib().kc_layer_norm_backward_workspace(desc, n))
    return n.value


def layer_norm_backward(desc: LayerNormDesc, d_x: int, d_mask: int, d_weight: int, d_stats: int, d_dy: int, d_dx: int,
                        d_dweight: int = 0, d_dbias: int = 0, d_workspace: int = 0, workspace_bytes: int = 0,
                        stream: int = 0):
    """kc_layer_norm_backward on device pointers: the gradients by x, weight and bias."""
    _check(lib().kc_layer_norm_backward(desc, d_x, d_mask, d_weight, d_stats, d_dy, d_dx, d_dweight, d_dbias,
                                        d_workspace, workspace_bytes, stream))


def embed_rows(desc: EmbedDesc, d_ids: int, d_table: int, d_x: int, d_y: int, stream: int = 0):
    """kc_embed_rows on device pointers: y[t] = x[t] + scale * table[id[t]] (d_x 0: no x)."""
    _check(lib().kc_embed_rows(desc, d_ids, d_table, d_x, d_y, stream))


def embed_rows_backward_workspace(desc: EmbedDesc) -> int:
    """kc_embed_rows_backward_workspace: bytes of device workspace a backward call needs."""
    n = ctypes.c_size_t()
    _check(lib().kc_embed_rows_backward_workspace(desc, n))
    return n.value


def embed_rows_backward(desc: EmbedDesc, d_ids: int, d_dy: int, d_dtable: int, d_workspace: int = 0,
                        workspace_bytes: int = 0, stream: int = 0):
    """kc_embed_rows_backward on device pointers: the table's gradient, float32."""
    _check(lib().kc_embed_rows_backward(desc, d_ids, d_dy, d_dtable, d_workspace, workspace_bytes, stream))


def distill_top(desc: DistillDesc, d_logits: int, d_ids: int, d_top_logits: int, d_teacher_log_sum: int, d_loss: int,
                d_stats: int = 0, stream: int = 0):
    """kc_distill_top on device pointers: each row's loss against a teacher's top logits (0 = not given)."""
    _check(lib().kc_distill_top(desc, d_logits, d_ids, d_top_logits, d_teacher_log_sum, d_loss, d_stats, stream))


def distill_top_backward(desc: DistillDesc, d_logits: int, d_ids: int, d_top_logits: int, d_teacher_log_sum: int,
                         d_stats: int, d_dloss: int, d_dlogits: int, stream: int = 0):
    """kc_distill_top_backward on device pointers: the gradient by the logits (d_dloss 0: 1 for every row)."""
    _check(lib().kc_distill_top_backward(desc, d_logits, d_ids, d_top_logits, d_teacher_log_sum, d_stats, d_dloss,
                                         d_dlogits, stream))


def pack_spatial(planes: np.ndarray) -> np.ndarray:
    """kc_pack_spatial: float planes [C, 19, 19] of 0 / 1 -> [C, PACKED_WORDS_PER_PLANE] uint32."""
    planes = np.ascontiguousarray(planes, np.float32)
    c = planes.shape[0]
    out = np.zeros((c, PACKED_WORDS_PER_PLANE), np.uint32)
    _check(lib().kc_pack_spatial(_fp(planes), c, out.ctypes.data_as(ctypes.POINTER(ctypes.c_uint32))))
    return out


def symmetry_table(symmetry: int, reverse: bool) -> np.ndarray:
    t = np.zeros(361, np.int32)
    _check(lib().kc_symmetry_table(symmetry, int(reverse), t.ctypes.data_as(ctypes.POINTER(I))))
    return t


def copy_with_symmetry(src: np.ndarray, n: int, h: int, w: int, c: int, symmetry: int, reverse: bool) -> np.ndarray:
    src = np.ascontiguousarray(src, np.float32)
    dst = np.zeros_like(src)
    _check(lib().kc_copy_with_symmetry(_fp(src), _fp(dst), n, h, w, c, symmetry, int(reverse)))
    return dst
