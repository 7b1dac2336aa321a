"""ctypes binding of libq3h (include/q3h.h) and a host mirror of the reference's
stack adapter.

`QwenLm` mirrors TQwenLm of src/tts/mormot.ai.tts.qwen.lm.pas:104-143
(Create / Reset / Forward / Length); `Talker` drives the device-resident
frame step that restates TQwenTalker.Start / NextFrame
(src/tts/mormot.ai.tts.qwen.talker.pas:471-681). Errors raise Q3HError with the
library's message, as the Pascal binding raises EQwenLm (lm.pas:41).

The library must be built (see __graft_entry__.build); nothing here falls back
to a CPU path: loading fails loudly when libq3h.so is missing.
"""
import ctypes
import os
import struct

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libq3h.so")

F32 = 0
Q8_0 = 1
BF16 = 2

# formats of a K/V cache (Q3H_KV_*)
KV_F32, KV_F16, KV_Q8, KV_Q4 = 0, 1, 2, 4
# rotary scalings (Q3H_ROPE_*)
ROPE_SCALING = {"plain": 0, "linear": 1, "yarn": 2, "bands": 3}
TREE_MAX_ROWS = 64  # Q3H_TREE_MAX_ROWS
TOP_MAX = 64  # Q3H_TOP_MAX

E_ARG, E_HIP, E_CAPACITY, E_STATE, E_NODEV = -1, -2, -3, -4, -5
NOALLOC_MAX_ROWS = 64  # Q3H_NOALLOC_MAX_ROWS
NOALLOC_SCRATCH_BYTES = 16 << 20  # Q3H_NOALLOC_SCRATCH_BYTES


class Q3HError(RuntimeError):
    def __init__(self, code, msg):
        super().__init__(f"q3h error {code}: {msg}")
        self.code = code


class StackConfig(ctypes.Structure):
    _fields_ = [
        ("layers", ctypes.c_int32),
        ("hidden", ctypes.c_int32),
        ("heads", ctypes.c_int32),
        ("kv_heads", ctypes.c_int32),
        ("head_dim", ctypes.c_int32),
        ("intermediate", ctypes.c_int32),
        ("rms_eps", ctypes.c_float),
        ("rope_theta", ctypes.c_float),
        ("dtype", ctypes.c_int32),
        ("kv_f16", ctypes.c_int32),
        ("act_q8", ctypes.c_int32),
        ("max_positions", ctypes.c_int32),
    ]


class LayerWeights(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in
                ("wq", "wk", "wv", "wo", "wgate", "wup", "wdown",
                 "input_norm", "post_norm", "q_norm", "k_norm")]


class Weights(ctypes.Structure):
    _fields_ = [
        ("src_dtype", ctypes.c_int32),
        ("layers", ctypes.POINTER(LayerWeights)),
        ("final_norm", ctypes.c_void_p),
    ]


class FrameConfig(ctypes.Structure):
    _fields_ = [
        ("n_streams", ctypes.c_int32),
        ("talker_head", ctypes.c_int32),
        ("cp_heads", ctypes.c_int32 * 15),
        ("vocab", ctypes.c_int32),
        ("cp_vocab", ctypes.c_int32),
        ("groups", ctypes.c_int32),
        ("eos", ctypes.c_int32),
        ("repetition_penalty", ctypes.c_float),
        ("max_frames", ctypes.c_int32),
        ("max_positions", ctypes.c_int32),
        ("use_graph", ctypes.c_int32),
    ]


class TextConfig(ctypes.Structure):
    _fields_ = [
        ("text_vocab", ctypes.c_int32),
        ("text_hidden", ctypes.c_int32),
        ("hidden", ctypes.c_int32),
        ("emb_dtype", ctypes.c_int32),
    ]


class Sampling(ctypes.Structure):
    _fields_ = [
        ("do_sample", ctypes.c_int32), ("temperature", ctypes.c_float),
        ("top_k", ctypes.c_int32), ("top_p", ctypes.c_float),
        ("sub_do_sample", ctypes.c_int32), ("sub_temperature", ctypes.c_float),
        ("sub_top_k", ctypes.c_int32), ("sub_top_p", ctypes.c_float),
        ("seed", ctypes.c_uint64),
    ]


class CodecRes(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in
                ("a1_alpha", "a1_beta", "c1_w", "c1_b", "a2_alpha", "a2_beta", "c2_w", "c2_b")]


class CodecBlock(ctypes.Structure):
    _fields_ = [("act_alpha", ctypes.c_void_p), ("act_beta", ctypes.c_void_p),
                ("up_w", ctypes.c_void_p), ("up_b", ctypes.c_void_p), ("res", CodecRes * 3)]


class CodecWeights(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p * 2) for n in
                ("up_w", "up_b", "dw_w", "dw_b", "norm_w", "norm_b", "pw1_w", "pw1_b", "pw2_w",
                 "pw2_b", "gamma")] + [
        ("conv0_w", ctypes.c_void_p), ("conv0_b", ctypes.c_void_p), ("block", CodecBlock * 4),
        ("out_alpha", ctypes.c_void_p), ("out_beta", ctypes.c_void_p),
        ("out_w", ctypes.c_void_p), ("out_b", ctypes.c_void_p)]


class StartIds(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int32) for n in
                ("tts_bos", "tts_eos", "tts_pad", "codec_pad", "codec_bos")]


class RopeConfig(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int32) for n in
                ("head_dim", "rot_dim", "interleaved", "max_positions")] + [
        ("theta", ctypes.c_float), ("scaling", ctypes.c_int32), ("factor", ctypes.c_float),
        ("original_positions", ctypes.c_int32), ("beta_fast", ctypes.c_float),
        ("beta_slow", ctypes.c_float), ("low_turns", ctypes.c_float),
        ("high_turns", ctypes.c_float), ("magnitude", ctypes.c_float)]


class CacheConfig(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int32) for n in
                ("sequences", "layers", "kv_heads", "head_dim", "max_positions", "format")]


class PagedConfig(ctypes.Structure):
    _fields_ = [("cache", CacheConfig), ("pages", ctypes.c_int32),
                ("page_positions", ctypes.c_int32)]


# q3h_append_args, q3h_attend_args and q3h_score_args, field by field in the
# header's order with C's alignment: packed for each call, which takes a quarter of
# the time that a ctypes structure does (2 us of a call's 8)
APPEND_ARGS = struct.Struct("4i3P3qPqPPfPPPP")
ATTEND_ARGS = struct.Struct("5ifPqPqPPPPq")
SCORE_ARGS = struct.Struct("Pq5iPPPPPPq")


class RowScores(ctypes.Structure):
    _fields_ = [("tokens_per_row", ctypes.c_int32), ("top_k", ctypes.c_int32)] + \
        [(n, ctypes.c_void_p) for n in
         ("tokens", "logprobs", "entropy", "top_ids", "top_logprobs")]


_P = ctypes.c_void_p
_I = ctypes.c_int
_FP = ctypes.POINTER(ctypes.c_float)
_IP = ctypes.POINTER(ctypes.c_int32)

# name -> (restype, argtypes): every entry point of include/q3h.h
SIGNATURES = {
    "q3h_device_available": (_I, []),
    "q3h_device_open": (_I, [_I, ctypes.POINTER(_P)]),
    "q3h_device_name": (ctypes.c_char_p, [_P]),
    "q3h_device_bytes": (ctypes.c_int64, [_P]),
    "q3h_device_close": (_I, [_P]),
    "q3h_last_error": (ctypes.c_char_p, []),
    "q3h_stack_create": (_I, [_P, ctypes.POINTER(StackConfig), ctypes.POINTER(Weights),
                              ctypes.POINTER(_P)]),
    "q3h_stack_add_head": (_I, [_P, _P, _I, _I, ctypes.POINTER(_I)]),
    "q3h_stack_bytes": (ctypes.c_int64, [_P]),
    "q3h_stack_destroy": (_I, [_P]),
    "q3h_context_create": (_I, [_P, _I, ctypes.POINTER(_P)]),
    "q3h_context_reset": (_I, [_P]),
    "q3h_context_length": (_I, [_P]),
    "q3h_context_destroy": (_I, [_P]),
    "q3h_context_fill_kv": (_I, [_P, _FP, _FP, _I]),
    "q3h_context_read_kv": (_I, [_P, _I, _FP, _FP]),
    "q3h_context_time_attention": (_I, [_P, _I, _FP, ctypes.POINTER(ctypes.c_int64)]),
    "q3h_forward_embeds": (_I, [_P, _FP, _I, _I, _FP, _FP]),
    "q3h_forward_embeds_noalloc": (_I, [_P, _FP, _I, _I, _FP, _FP]),
    "q3h_forward_embeds_probe": (_I, [_P, _FP, _I, _I, _FP, _FP, _FP, _FP]),
    "q3h_forward_embeds_batch": (_I, [ctypes.POINTER(_P), _I, _FP, _IP, _FP, _FP]),
    "q3h_frame_create": (_I, [_P, _P, ctypes.POINTER(FrameConfig), _FP,
                              ctypes.POINTER(_FP), _FP, ctypes.POINTER(_P)]),
    "q3h_frame_start": (_I, [_P, _I, _FP, _I, _FP, _I]),
    "q3h_frame_start_batch": (_I, [_P, _I, ctypes.POINTER(ctypes.c_int),
                                   ctypes.POINTER(_FP), ctypes.POINTER(ctypes.c_int),
                                   ctypes.POINTER(_FP), ctypes.POINTER(ctypes.c_int)]),
    "q3h_frame_step": (_I, [_P, _IP, _IP]),
    "q3h_frame_state": (_I, [_P, _I, _FP, _FP]),
    "q3h_frame_destroy": (_I, [_P]),
    "q3h_text_create": (_I, [_P, ctypes.POINTER(TextConfig), _P, _FP, _FP, _FP, _FP,
                             ctypes.POINTER(_P)]),
    "q3h_text_project": (_I, [_P, _IP, _I, _FP]),
    "q3h_text_destroy": (_I, [_P]),
    "q3h_frame_set_sampling": (_I, [_P, ctypes.POINTER(Sampling)]),
    "q3h_codec_create": (_I, [_P, ctypes.POINTER(CodecWeights), _I, ctypes.POINTER(_P)]),
    "q3h_codec_reset": (_I, [_P]),
    "q3h_codec_back": (_I, [_P, _FP, _I, _FP]),
    "q3h_codec_bytes": (ctypes.c_int64, [_P]),
    "q3h_codec_destroy": (_I, [_P]),
    "q3h_frame_start_text": (_I, [_P, _I, _P, ctypes.POINTER(StartIds), _IP, _I, _IP, _I, _I]),
    "q3h_rope_create": (_I, [_P, ctypes.POINTER(RopeConfig), ctypes.POINTER(_P)]),
    "q3h_rope_create_axes": (_I, [_P, ctypes.POINTER(RopeConfig), _I, _IP, ctypes.POINTER(_P)]),
    "q3h_rope_destroy": (_I, [_P]),
    "q3h_cache_create": (_I, [_P, ctypes.POINTER(CacheConfig), ctypes.POINTER(_P)]),
    "q3h_cache_create_paged": (_I, [_P, ctypes.POINTER(PagedConfig), ctypes.POINTER(_P)]),
    "q3h_cache_bytes": (ctypes.c_int64, [_P]),
    "q3h_cache_destroy": (_I, [_P]),
    "q3h_cache_append": (_I, [_P, _P, _P]),
    "q3h_cache_append_at": (_I, [_P, _P, _P, _P]),
    "q3h_cache_read": (_I, [_P, _I, _I, _I, _P, _P, _P, _P, _P]),
    "q3h_cache_attend_workspace": (ctypes.c_int64, [_P, _I, _I, _I, _I]),
    "q3h_cache_attend": (_I, [_P, _P, _P]),
    "q3h_cache_keep": (_I, [_P, _I, _I, _P, _P, _P, _P]),
    "q3h_cache_reserve": (_I, [_P, _I, _I, _P, _P, _P, _P]),
    "q3h_cache_fork": (_I, [_P, _I, _P, _P, _P]),
    "q3h_cache_release": (_I, [_P, _I, _P, _P]),
    "q3h_cache_compact": (_I, [_P, _P, _P]),
    "q3h_cache_copy": (_I, [_P, _P, _I, _P, _P, _P]),
    "q3h_cache_page_state": (_I, [_P, _P, _P, _P, _P]),
    "q3h_token_logprobs_workspace": (ctypes.c_int64, [_I, _I, _I]),
    "q3h_token_logprobs": (_I, [_P, _P, _P]),
    "q3h_stack_set_rope": (_I, [_P, ctypes.POINTER(RopeConfig)]),
    "q3h_forward_tree": (_I, [_P, _FP, _I, _IP, _I, ctypes.POINTER(RowScores), _FP, _FP]),
    "q3h_context_keep": (_I, [_P, _IP, _I]),
    "q3h_forward_score": (_I, [_P, _FP, _I, _I, ctypes.POINTER(RowScores), _FP, _FP]),
    "q3h_quantize_row_q8_0": (_I, [_FP, _P, ctypes.c_int64]),
    "q3h_stack_time_gemv": (_I, [_P, _I, _I, _I, _FP, ctypes.POINTER(_I),
                                 ctypes.POINTER(ctypes.c_int64)]),
}

_lib = None


def lib():
    """The loaded libq3h (raises if it was not built)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise OSError(f"{LIB_PATH} is missing: build it with __graft_entry__.build()")
        L = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(L, name)
            fn.restype = res
            fn.argtypes = args
        _lib = L
    return _lib


def _check(rc):
    if rc != 0:
        raise Q3HError(rc, lib().q3h_last_error().decode(errors="replace"))


def _fp(a):
    return a.ctypes.data_as(_FP) if a is not None else None


def _f32(a):
    return np.ascontiguousarray(a, dtype=np.float32)


def available():
    return bool(lib().q3h_device_available())


def quantize_q8_0(x):
    """ggml quantize_row_q8_0_ref of a float32 matrix [..., k]: uint8 blocks."""
    x = _f32(x)
    k = x.size
    out = np.empty(k // 32 * 34, dtype=np.uint8)
    _check(lib().q3h_quantize_row_q8_0(_fp(x), out.ctypes.data_as(_P), k))
    return out.reshape(x.shape[:-1] + (x.shape[-1] // 32 * 34,))


class Device:
    """TQwenVulkan (lm.pas:44-62) for a gfx950 device."""

    def __init__(self, ordinal=0):
        h = _P()
        _check(lib().q3h_device_open(ordinal, ctypes.byref(h)))
        self.h = h
        self.ordinal = ordinal

    @property
    def name(self):
        return lib().q3h_device_name(self.h).decode()

    @property
    def bytes(self):
        return lib().q3h_device_bytes(self.h)

    def close(self):
        if self.h:
            _check(lib().q3h_device_close(self.h))
            self.h = None


class Stack:
    """A Qwen3 stack on the device (TQwen3Model.CreateStack + TQwen3Vulkan.Create)."""

    def __init__(self, dev, cfg, layers, final_norm, src_dtype):
        """cfg: dict of StackConfig fields; layers: list of dicts with wq..wdown
        (float32 [out][in] or uint8 Q8_0 blocks [out][in/32*34]) and the norm
        vectors; src_dtype: F32 or Q8_0."""
        self.cfg = dict(cfg)
        c = StackConfig(**{k: cfg[k] for k, _ in StackConfig._fields_})
        keep = []
        arr = (LayerWeights * len(layers))()
        for i, L in enumerate(layers):
            for name in ("wq", "wk", "wv", "wo", "wgate", "wup", "wdown"):
                a = np.ascontiguousarray(L[name])
                keep.append(a)
                setattr(arr[i], name, a.ctypes.data)
            for name in ("input_norm", "post_norm", "q_norm", "k_norm"):
                a = _f32(L[name])
                keep.append(a)
                setattr(arr[i], name, a.ctypes.data)
        fn = _f32(final_norm)
        w = Weights(src_dtype, arr, fn.ctypes.data)
        h = _P()
        _check(lib().q3h_stack_create(dev.h, ctypes.byref(c), ctypes.byref(w), ctypes.byref(h)))
        self.h = h
        self.head_rows = []

    def add_head(self, w, src_dtype):
        a = np.ascontiguousarray(w)
        rows = a.shape[0]
        idx = ctypes.c_int()
        _check(lib().q3h_stack_add_head(self.h, a.ctypes.data_as(_P), rows, src_dtype,
                                        ctypes.byref(idx)))
        self.head_rows.append(rows)
        return idx.value

    def set_rope(self, theta, rot_dim=None, interleaved=False, scaling=None, magnitude=0.0):
        """Rotary positions of every context made from now on (as Rope's)."""
        cfg = _rope_config(self.cfg["head_dim"], self.cfg["max_positions"], theta, rot_dim,
                           interleaved, scaling, magnitude)
        _check(lib().q3h_stack_set_rope(self.h, ctypes.byref(cfg)))

    @property
    def bytes(self):
        return lib().q3h_stack_bytes(self.h)

    def time_gemv(self, head=-1, iters=20, mode=1):
        """(us per launch, launches per step, algorithmic bytes per step) of the
        weight products of one single-row decode step. mode 0: direct launches,
        wall time; 1: hipGraph replay, wall time; 2: the kernels' own execution
        time (events attached to each launch)."""
        us = ctypes.c_float()
        n = ctypes.c_int()
        b = ctypes.c_int64()
        _check(lib().q3h_stack_time_gemv(self.h, head, iters, int(mode), ctypes.byref(us),
                                         ctypes.byref(n), ctypes.byref(b)))
        return us.value, n.value, b.value

    def destroy(self):
        if self.h:
            _check(lib().q3h_stack_destroy(self.h))
            self.h = None


class Context:
    """A K/V cache of a stack (NewContext / TDecoderContext)."""

    def __init__(self, stack, max_positions):
        h = _P()
        _check(lib().q3h_context_create(stack.h, max_positions, ctypes.byref(h)))
        self.h = h
        self.stack = stack

    def reset(self):
        _check(lib().q3h_context_reset(self.h))

    @property
    def length(self):
        n = lib().q3h_context_length(self.h)
        if n < 0:
            _check(n)
        return n

    def forward(self, x, head=-1, want_logits=True, want_normed=True, noalloc=False):
        """x [rows][hidden]; returns (logits or None, normed_last or None).
        noalloc: through q3h_forward_embeds_noalloc (work buffers in the
        device's static scratch array, at most NOALLOC_MAX_ROWS rows)."""
        x = _f32(x)
        if x.ndim == 1:
            x = x[None, :]
        rows, hidden = x.shape
        logits = None
        if 0 <= head < len(self.stack.head_rows) and want_logits:
            logits = np.empty(self.stack.head_rows[head], dtype=np.float32)
        normed = np.empty(hidden, dtype=np.float32) if want_normed else None
        # an unknown head index goes to the library, which reports it
        fn = lib().q3h_forward_embeds_noalloc if noalloc else lib().q3h_forward_embeds
        _check(fn(self.h, _fp(x), rows, head, _fp(logits), _fp(normed)))
        return logits, normed

    def forward_probe(self, x, head=-1):
        """forward() with the probe of TQwenLm (lm.pas:380-389): returns
        (logits or None, normed_last, layer_out [layers][rows][hidden],
        normed_rows [rows][hidden]): every layer's output ("name.layerN") and
        the final-normed state of every row ("name.out")."""
        x = _f32(x)
        if x.ndim == 1:
            x = x[None, :]
        rows, hidden = x.shape
        logits = None
        if 0 <= head < len(self.stack.head_rows):
            logits = np.empty(self.stack.head_rows[head], dtype=np.float32)
        normed = np.empty(hidden, dtype=np.float32)
        lo = np.empty((self.stack.cfg["layers"], rows, hidden), dtype=np.float32)
        nr = np.empty((rows, hidden), dtype=np.float32)
        _check(lib().q3h_forward_embeds_probe(self.h, _fp(x), rows, head, _fp(logits),
                                              _fp(normed), _fp(lo), _fp(nr)))
        return logits, normed, lo, nr

    def _scored(self, rows, head, tokens, top_k):
        """(the structure of a call's scores, their arrays by name)."""
        t = np.zeros((rows, 0), np.int32) if tokens is None else \
            np.ascontiguousarray(tokens, dtype=np.int32)
        if t.ndim == 1:
            t = t[:, None]
        if t.ndim != 2 or t.shape[0] != rows:
            _bad(f"tokens are {list(t.shape)}, not of {rows} rows")
        res = {"logprobs": np.empty(t.shape, np.float32), "entropy": np.empty(rows, np.float32)}
        sc = RowScores(t.shape[1], top_k, t.ctypes.data, res["logprobs"].ctypes.data,
                       res["entropy"].ctypes.data)
        if top_k > 0:
            res["top_ids"] = np.empty((rows, top_k), np.int32)
            res["top_logprobs"] = np.empty((rows, top_k), np.float32)
            sc.top_ids = res["top_ids"].ctypes.data
            sc.top_logprobs = res["top_logprobs"].ctypes.data
        sc.keep = t
        return sc, res

    def _all_rows(self, x, head, tokens, top_k, want_logits, want_normed, want_scores, call):
        x = _f32(x)
        if x.ndim != 2 or x.shape[1] != self.stack.cfg["hidden"]:
            _bad(f"x is {list(x.shape)}, not [rows][{self.stack.cfg['hidden']}]")
        rows, hidden = x.shape
        known = 0 <= head < len(self.stack.head_rows)
        logits = np.empty((rows, self.stack.head_rows[head]), np.float32) \
            if known and want_logits else None
        normed = np.empty((rows, hidden), np.float32) if want_normed else None
        sc, res = self._scored(rows, head, tokens, top_k) if want_scores else (None, {})
        _check(call(x, rows, ctypes.byref(sc) if sc is not None else None, logits, normed))
        if logits is not None:
            res["logits"] = logits
        if normed is not None:
            res["normed"] = normed
        return res

    def forward_tree(self, x, parents, head=-1, tokens=None, top_k=0, want_logits=True,
                     want_normed=True, want_scores=False):
        """A tree of drafted rows x [rows][hidden], row r after row parents[r] (-1:
        after the context's last position): dict of logits [rows][head rows],
        normed [rows][hidden] and, with want_scores, those of token_logprobs (of
        tokens [rows][m]). The length stays; keep() takes a path of them over."""
        p = np.ascontiguousarray(parents, dtype=np.int32)
        if p.shape != (len(x),):
            _bad(f"{list(p.shape)} parents of {len(x)} rows")
        return self._all_rows(
            x, head, tokens, top_k, want_logits, want_normed, want_scores,
            lambda a, n, sc, lg, nm: lib().q3h_forward_tree(
                self.h, _fp(a), n, p.ctypes.data_as(_IP), head, sc, _fp(lg), _fp(nm)))

    def keep(self, kept):
        """The rows kept of the last forward_tree, a path from a root down, become
        the context's next positions."""
        k = np.ascontiguousarray(kept, dtype=np.int32)
        _check(lib().q3h_context_keep(self.h, k.ctypes.data_as(_IP), len(k)))

    def forward_score(self, x, head, tokens=None, top_k=0, want_logits=False, want_normed=False):
        """forward() of rows x, every position scored: dict as token_logprobs gives
        it (of tokens [rows][m]), with logits and normed of every row when wanted."""
        return self._all_rows(
            x, head, tokens, top_k, want_logits, want_normed, True,
            lambda a, n, sc, lg, nm: lib().q3h_forward_score(
                self.h, _fp(a), n, head, sc, _fp(lg), _fp(nm)))

    def fill_kv(self, k, v):
        """k, v: float32 [layers][kv_heads][len][head_dim]."""
        k, v = _f32(k), _f32(v)
        _check(lib().q3h_context_fill_kv(self.h, _fp(k), _fp(v), k.shape[2]))

    def time_attention(self, iters=20):
        """(us per launch, algorithmic bytes per launch) of the decode attention
        of one new row at position length, averaged over the layers and iters
        (events attached to each launch); the length does not change."""
        us = ctypes.c_float()
        b = ctypes.c_int64()
        _check(lib().q3h_context_time_attention(self.h, iters, ctypes.byref(us), ctypes.byref(b)))
        return us.value, b.value

    def read_kv(self, layer):
        c = self.stack.cfg
        n = self.length
        k = np.empty((c["kv_heads"], n, c["head_dim"]), dtype=np.float32)
        v = np.empty_like(k)
        _check(lib().q3h_context_read_kv(self.h, layer, _fp(k), _fp(v)))
        return k, v

    def destroy(self):
        if self.h:
            _check(lib().q3h_context_destroy(self.h))
            self.h = None


def forward_batch(ctxs, x, heads=None, want_normed=True):
    """One row per context: x [n][hidden]; heads: list of head indices or None."""
    x = _f32(x)
    n, hidden = x.shape
    arr = (_P * n)(*[c.h.value for c in ctxs])
    logits = None
    hp = None
    if heads is not None:
        ha = np.ascontiguousarray(heads, dtype=np.int32)
        hp = ha.ctypes.data_as(_IP)
        logits = np.empty((n, ctxs[0].stack.head_rows[heads[0]]), dtype=np.float32)
    normed = np.empty((n, hidden), dtype=np.float32) if want_normed else None
    _check(lib().q3h_forward_embeds_batch(arr, n, _fp(x), hp, _fp(logits), _fp(normed)))
    return logits, normed


class QwenLm:
    """TQwenLm (lm.pas:104-143): one stack, its heads, one context.

    forward(x, rows, output) follows TQwenLm.Forward (lm.pas:391-408): the rows
    are appended at positions length..length+rows-1, the normed state of the
    last row and the logits of head `output` come back."""

    def __init__(self, stack, max_positions):
        self.stack = stack
        self.ctx = Context(stack, max_positions)
        self.length = 0

    def reset(self):
        self.ctx.reset()
        self.length = 0

    def forward(self, x, output=-1):
        x = _f32(x)
        rows = 1 if x.ndim == 1 else x.shape[0]
        if rows <= 0:
            return None, None
        logits, hidden = self.ctx.forward(x, output)
        self.length += rows
        return logits, hidden

    def destroy(self):
        self.ctx.destroy()


class TextProj:
    """The talker's text projection on the device (TQwenTalker.TextProject,
    talker.pas:390-421): emb float32 [vocab][text_hidden] or uint16 (the BF16
    bits), fc1 [text_hidden][text_hidden], fc2 [hidden][text_hidden] + biases."""

    def __init__(self, dev, emb, fc1_w, fc1_b, fc2_w, fc2_b):
        emb = np.ascontiguousarray(emb)
        dt = BF16 if emb.dtype == np.uint16 else F32
        if dt == F32:
            emb = _f32(emb)
        self._w = [_f32(fc1_w), _f32(fc1_b), _f32(fc2_w), _f32(fc2_b)]
        cfg = TextConfig(emb.shape[0], emb.shape[1], self._w[2].shape[0], dt)
        h = _P()
        _check(lib().q3h_text_create(dev.h, ctypes.byref(cfg), emb.ctypes.data_as(_P),
                                     *[_fp(a) for a in self._w], ctypes.byref(h)))
        self._w = None
        self.h = h
        self.hidden = cfg.hidden

    def project(self, ids):
        ids = np.ascontiguousarray(ids, dtype=np.int32)
        y = np.empty((len(ids), self.hidden), dtype=np.float32)
        _check(lib().q3h_text_project(self.h, ids.ctypes.data_as(_IP), len(ids), _fp(y)))
        return y

    def destroy(self):
        if self.h:
            _check(lib().q3h_text_destroy(self.h))
            self.h = None


class Codec:
    """The back part of the 12 Hz decoder on the device (TQwenCodecVulkan:
    Back / Reset, codec.vulkan.pas:455-488, 633-652). w: dict of the
    decoder.* tensors (f32, safetensors layouts; see synth.codec_weights)."""

    def __init__(self, dev, w, max_frames=16):
        keep = []

        def ptr(a):
            if a is None:
                return None  # NULL: the library reports the missing tensor
            a = np.ascontiguousarray(a, dtype=np.float32)
            keep.append(a)
            return a.ctypes.data

        s = CodecWeights()
        for name in ("up_w", "up_b", "dw_w", "dw_b", "norm_w", "norm_b", "pw1_w", "pw1_b",
                     "pw2_w", "pw2_b", "gamma"):
            arr = getattr(s, name)
            for i in range(2):
                arr[i] = ptr(w[name][i])
        s.conv0_w, s.conv0_b = ptr(w["conv0_w"]), ptr(w["conv0_b"])
        for i, b in enumerate(w["block"]):
            blk = s.block[i]
            blk.act_alpha, blk.act_beta = ptr(b["act_alpha"]), ptr(b["act_beta"])
            blk.up_w, blk.up_b = ptr(b["up_w"]), ptr(b["up_b"])
            for r, rw in enumerate(b["res"]):
                for k, v in rw.items():
                    setattr(blk.res[r], k, ptr(v))
        s.out_alpha, s.out_beta = ptr(w["out_alpha"]), ptr(w["out_beta"])
        s.out_w, s.out_b = ptr(w["out_w"]), ptr(w["out_b"])
        h = _P()
        _check(lib().q3h_codec_create(dev.h, ctypes.byref(s), max_frames, ctypes.byref(h)))
        self.h = h

    def back(self, x):
        """x [frames][1024] -> pcm [frames * 1920]."""
        x = _f32(x)
        frames = x.shape[0]
        pcm = np.empty(frames * 1920, dtype=np.float32)
        _check(lib().q3h_codec_back(self.h, _fp(x), frames, _fp(pcm)))
        return pcm

    def reset(self):
        _check(lib().q3h_codec_reset(self.h))

    @property
    def bytes(self):
        return lib().q3h_codec_bytes(self.h)

    def destroy(self):
        if self.h:
            _check(lib().q3h_codec_destroy(self.h))
            self.h = None


class Frame:
    """The device-resident frame step over n streams (q3h_frame_*)."""

    def __init__(self, talker, cp, codec_emb, pred_emb, tts_pad, n_streams=1, talker_head=0,
                 cp_heads=None, eos=-1, penalty=1.05, max_frames=256, max_positions=1024,
                 use_graph=True, groups=16):
        vocab, hidden = codec_emb.shape
        cp_vocab = pred_emb[0].shape[0]
        cfg = FrameConfig()
        cfg.n_streams = n_streams
        cfg.talker_head = talker_head
        heads = list(cp_heads) if cp_heads is not None else list(range(groups - 1))
        for i in range(15):
            cfg.cp_heads[i] = heads[i] if i < len(heads) else 0
        cfg.vocab = vocab
        cfg.cp_vocab = cp_vocab
        cfg.groups = groups
        cfg.eos = eos
        cfg.repetition_penalty = penalty
        cfg.max_frames = max_frames
        cfg.max_positions = max_positions
        cfg.use_graph = 1 if use_graph else 0
        self.cfg = cfg
        ce = _f32(codec_emb)
        pe = [_f32(p) for p in pred_emb]
        pa = (_FP * len(pe))(*[_fp(p) for p in pe])
        tp = _f32(tts_pad)
        h = _P()
        _check(lib().q3h_frame_create(talker.h, cp.h, ctypes.byref(cfg), _fp(ce), pa, _fp(tp),
                                      ctypes.byref(h)))
        self.h = h
        self.n = n_streams
        self.groups = groups
        self.vocab = vocab
        self.hidden = hidden

    def start(self, stream, prefill, trailing=None):
        p = _f32(prefill)
        t = _f32(trailing) if trailing is not None and len(trailing) else None
        _check(lib().q3h_frame_start(self.h, stream, _fp(p), p.shape[0], _fp(t),
                                     0 if t is None else t.shape[0]))

    def start_batch(self, streams, prefills, trailings=None):
        """q3h_frame_start_batch: the starts of several streams at once, their
        prefills overlapping on the device (prefills[i] [rows][hidden],
        trailings[i] None or [rows][hidden])."""
        n = len(streams)
        ps = [_f32(p) for p in prefills]
        ts = [None] * n if trailings is None else \
            [_f32(t) if t is not None and len(t) else None for t in trailings]
        c_streams = (ctypes.c_int * n)(*[int(x) for x in streams])
        c_pre = (_FP * n)(*[_fp(p) for p in ps])
        c_rows = (ctypes.c_int * n)(*[p.shape[0] for p in ps])
        c_tr = (_FP * n)(*[_fp(t) for t in ts])
        c_trr = (ctypes.c_int * n)(*[0 if t is None else t.shape[0] for t in ts])
        _check(lib().q3h_frame_start_batch(self.h, n, c_streams, c_pre, c_rows, c_tr, c_trr))

    def set_sampling(self, do_sample=False, temperature=1.0, top_k=0, top_p=1.0,
                     sub_do_sample=False, sub_temperature=1.0, sub_top_k=0, sub_top_p=1.0,
                     seed=0):
        """TQwenTalker.Sampling (talker.pas:150): the talker's and the code
        predictor's choosers; seed 0 draws a fresh sentence seed per start."""
        sp = Sampling(int(do_sample), temperature, top_k, top_p, int(sub_do_sample),
                      sub_temperature, sub_top_k, sub_top_p, seed)
        _check(lib().q3h_frame_set_sampling(self.h, ctypes.byref(sp)))

    def start_text(self, stream, proj, ids, codec, tts_bos, tts_eos, tts_pad, codec_pad,
                   codec_bos, non_streaming):
        """TQwenTalker.Start from token ids (talker.pas:471-593): the prefill
        and trailing rows built on the device with proj (a TextProj)."""
        sp = StartIds(tts_bos, tts_eos, tts_pad, codec_pad, codec_bos)
        a = np.ascontiguousarray(ids, dtype=np.int32)
        c = np.ascontiguousarray(codec, dtype=np.int32)
        _check(lib().q3h_frame_start_text(self.h, stream, proj.h, ctypes.byref(sp),
                                          a.ctypes.data_as(_IP), len(a),
                                          c.ctypes.data_as(_IP), len(c),
                                          1 if non_streaming else 0))

    def step(self):
        codes = np.empty((self.n, self.groups), dtype=np.int32)
        alive = np.empty(self.n, dtype=np.int32)
        _check(lib().q3h_frame_step(self.h, codes.ctypes.data_as(_IP),
                                    alive.ctypes.data_as(_IP)))
        return codes, alive

    def state(self, stream):
        logits = np.empty(self.vocab, dtype=np.float32)
        past = np.empty(self.hidden, dtype=np.float32)
        _check(lib().q3h_frame_state(self.h, stream, _fp(logits), _fp(past)))
        return logits, past

    def destroy(self):
        if self.h:
            _check(lib().q3h_frame_destroy(self.h))
            self.h = None


# ---------------------------------------------------------------------------
# operators on device memory: torch tensors of the handle's device, in the order
# of torch's current stream there (no copies, no waits; they can be captured)


def _bad(msg):
    raise Q3HError(E_ARG, msg)


_torch = None


def _use_torch():
    """torch, imported with the first handle that takes its tensors."""
    global _torch
    if _torch is None:
        import torch
        _torch = torch
    return _torch


def _ptr(t, ordinal, dtype, name):
    """The address of a tensor of this dtype on the device."""
    if t.get_device() != ordinal:
        _bad(f"{name} is on {t.device}, not on device {ordinal}")
    if t.dtype is not dtype:
        _bad(f"{name} is {t.dtype}, not {dtype}")
    return t.data_ptr()


def _rows(t, n, rows, heads, hd, ordinal, name):
    """(address, floats between rows) of f32 rows [n][rows][heads][hd], or
    [n][rows][heads * hd], contiguous within a row."""
    shape, width = t.shape, heads * hd
    if shape != (n, rows, heads, hd) and shape != (n, rows, width):
        _bad(f"{name} is {list(shape)}, not {[n, rows, heads, hd]}")
    if t.get_device() != ordinal or t.dtype is not _torch.float32:
        _ptr(t, ordinal, _torch.float32, name)
    if t.is_contiguous():
        return t.data_ptr(), width
    stride = t.stride()
    if stride[-1] != 1 or (len(shape) == 4 and heads > 1 and stride[2] != hd):
        _bad(f"{name}: the heads of a row are not side by side")
    ld = stride[1] if rows > 1 else stride[0] if n > 1 else width
    if rows > 1 and n > 1 and stride[0] != rows * ld:
        _bad(f"{name}: the sequences' rows are not evenly spaced")
    return t.data_ptr(), ld


def _whole(t, shape, ordinal, dtype, name):
    """The address of a contiguous tensor of this shape and dtype; 0 for None."""
    if t is None:
        return 0
    if t.shape != shape or not t.is_contiguous():
        _bad(f"{name} is {list(t.shape)}, not contiguous {list(shape)}")
    if t.get_device() != ordinal or t.dtype is not dtype:
        _ptr(t, ordinal, dtype, name)
    return t.data_ptr()


def _stream(ordinal):
    return _torch._C._cuda_getCurrentRawStream(ordinal)


def _rope_config(head_dim, max_positions, theta, rot_dim, interleaved, scaling, magnitude):
    s = dict(scaling or {"kind": "plain"})
    kind = s.pop("kind")
    if kind not in ROPE_SCALING:
        _bad(f"no rotary scaling {kind!r}")
    cfg = RopeConfig(head_dim, head_dim if rot_dim is None else rot_dim, int(interleaved),
                     max_positions, theta, ROPE_SCALING[kind], s.pop("factor", 1.0),
                     s.pop("original", 0), s.pop("beta_fast", 32.0), s.pop("beta_slow", 1.0),
                     s.pop("low", 1.0), s.pop("high", 4.0), magnitude)
    if s:
        _bad(f"unknown rotary settings {sorted(s)}")
    return cfg


class Rope:
    """A rotary table (q3h_rope_*): the first rot_dim elements of a head turned
    in neighbouring pairs (interleaved) or in pairs half of them apart. scaling:
    None, dict(kind="linear", factor=), dict(kind="yarn", factor=, original=,
    beta_fast=32, beta_slow=1), dict(kind="bands", factor=, original=, low=1,
    high=4); magnitude: on cosine and sine (0: the scaling's own). axes: the axis of
    each pair (0 .. 3), whose positions Cache.append gets."""

    h = None

    def __init__(self, dev, head_dim, max_positions, theta, rot_dim=None, interleaved=False,
                 scaling=None, magnitude=0.0, axes=None):
        cfg = _rope_config(head_dim, max_positions, theta, rot_dim, interleaved, scaling,
                           magnitude)
        h = _P()
        L = lib()
        self.axes = 1
        if axes is None:
            _check(L.q3h_rope_create(dev.h, ctypes.byref(cfg), ctypes.byref(h)))
        else:
            pairs = [int(x) for x in axes]
            if len(pairs) != cfg.rot_dim // 2:
                _bad(f"axes of {len(pairs)} pairs, not of {cfg.rot_dim // 2}")
            if not all(0 <= x < 4 for x in pairs):  # (32 bits would make others of some)
                _bad(f"axes {sorted(set(pairs))}, not of 0 .. 3")
            self.axes = max(pairs, default=0) + 1
            _check(L.q3h_rope_create_axes(dev.h, ctypes.byref(cfg), self.axes,
                                          (ctypes.c_int32 * len(pairs))(*pairs), ctypes.byref(h)))
        self.dev = dev
        self.h = h
        self._destroy = L.q3h_rope_destroy

    def destroy(self):
        if self.h:
            _check(self._destroy(self.h))
            self.h = None

    def __del__(self):
        if self.h and self.dev.h:
            self._destroy(self.h)


class Cache:
    """A K/V cache of several sequences (q3h_cache_*), in f32, f16, one byte
    per element with a scale per position and head, or four bits with steps for each
    32 elements too (KV_F32, KV_F16, KV_Q8, KV_Q4). With pages: in that many pages of
    page_positions positions (32, 64, 128 or 256) that the sequences share (reserve,
    fork, release, compact). Calls take rows [sequences][rows][heads][head_dim] for the
    first sequences of the cache; lens, counts [sequences] and parents
    [sequences][rows] are int32 tensors on the device."""

    h = None

    def __init__(self, dev, sequences, kv_heads, head_dim, max_positions, fmt=KV_F32, layers=1,
                 pages=0, page_positions=64):
        cfg = CacheConfig(sequences, layers, kv_heads, head_dim, max_positions, fmt)
        h = _P()
        L = lib()
        _use_torch()
        self.dev = dev
        self._destroy = L.q3h_cache_destroy
        if pages:
            paged = PagedConfig(cfg, pages, page_positions)
            _check(L.q3h_cache_create_paged(dev.h, ctypes.byref(paged), ctypes.byref(h)))
        else:
            _check(L.q3h_cache_create(dev.h, ctypes.byref(cfg), ctypes.byref(h)))
        self.h = h  # (from here on __del__ gives it back)
        self.pages = pages
        self.table_shape = (sequences, -(-max_positions // page_positions)) if pages else None
        self.kv_heads, self.head_dim = kv_heads, head_dim
        self._append, self._read, self._attend = \
            L.q3h_cache_append, L.q3h_cache_read, L.q3h_cache_attend
        self._append_at = L.q3h_cache_append_at
        self._reserve, self._fork, self._release = \
            L.q3h_cache_reserve, L.q3h_cache_fork, L.q3h_cache_release
        self._compact, self._copy, self._page_state = \
            L.q3h_cache_compact, L.q3h_cache_copy, L.q3h_cache_page_state
        self._device = _torch.device("cuda", dev.ordinal)
        self._workspace = L.q3h_cache_attend_workspace

    @property
    def bytes(self):
        return lib().q3h_cache_bytes(self.h)

    def append(self, k, v, lens, counts=None, parents=None, q=None, q_out=None, rope=None,
               q_norm=None, k_norm=None, eps=1e-6, layer=0, positions=None):
        """Writes the drafted rows k, v at positions lens[b] + row, keys and
        queries normed (q_norm, k_norm) and turned (rope) first. Returns the
        queries (q_out, made when it is None; rows beyond counts as they were),
        None without q. parents: the row each row continues (-1: the sequence
        itself); None: a chain. positions [axes of the rope][sequences][rows]: those
        that the rows are turned by (None: lens[b] plus their depth)."""
        o, hd, i32, f32 = self.dev.ordinal, self.head_dim, _torch.int32, _torch.float32
        n, rows = k.shape[0], k.shape[1]
        pk, ldk = _rows(k, n, rows, self.kv_heads, hd, o, "k")
        pv, ldv = _rows(v, n, rows, self.kv_heads, hd, o, "v")
        heads = pq = ldq = po = ldo = qn = turn = 0
        if rope is not None:
            turn = rope.h.value if rope.h else _bad("the rotary table is destroyed")
        if q is not None:
            heads = q.shape[2] if q.dim() == 4 else q.shape[2] // hd
            if q_out is None:
                q_out = q.new_empty((n, rows, heads, hd))
            pq, ldq = _rows(q, n, rows, heads, hd, o, "q")
            po, ldo = _rows(q_out, n, rows, heads, hd, o, "q_out")
            qn = _whole(q_norm, (hd,), o, f32, "q_norm")
        a = APPEND_ARGS.pack(
            layer, n, rows, heads, pq, pk, pv, ldq, ldk, ldv, po, ldo, qn,
            _whole(k_norm, (hd,), o, f32, "k_norm"), eps, turn,
            _whole(lens, (n,), o, i32, "lens"), _whole(counts, (n,), o, i32, "counts"),
            _whole(parents, (n, rows), o, i32, "parents"))
        if positions is None:
            _check(self._append(self.h, a, _stream(o)))
        else:
            at = _whole(positions, (rope.axes if rope is not None else 1, n, rows), o, i32,
                        "positions")
            _check(self._append_at(self.h, a, at, _stream(o)))
        return q_out

    def read(self, k, v, starts=None, counts=None, layer=0):
        """Positions starts[b] .. + counts[b] - 1 of the first sequences into k
        and v (either None) [sequences][rows][kv_heads][head_dim] as f32; rows
        beyond counts stay as they were."""
        o, i32, f32 = self.dev.ordinal, _torch.int32, _torch.float32
        like = k if k is not None else v
        if like is None:
            _bad("neither k nor v")
        n, rows = like.shape[0], like.shape[1]
        shape = (n, rows, self.kv_heads, self.head_dim)
        _check(self._read(
            self.h, layer, n, rows, _whole(starts, (n,), o, i32, "starts"),
            _whole(counts, (n,), o, i32, "counts"), _whole(k, shape, o, f32, "k"),
            _whole(v, shape, o, f32, "v"), _stream(o)))

    def attend(self, q, lens, max_len, out=None, counts=None, parents=None, scale=0.0, layer=0,
               workspace=None):
        """Attention of the drafted rows q over the cache, which holds their keys
        and values already; max_len: no length in lens is above it. Returns out
        (made when it is None; rows beyond counts as they were). scale 0: 1 /
        sqrt(head_dim). workspace: a uint8 tensor of attend_workspace bytes (made
        when it is None)."""
        o, hd, i32 = self.dev.ordinal, self.head_dim, _torch.int32
        n, rows = q.shape[0], q.shape[1]
        heads = q.shape[2] if q.dim() == 4 else q.shape[2] // hd
        if out is None:
            out = q.new_empty((n, rows, heads, hd))
        pq, ldq = _rows(q, n, rows, heads, hd, o, "q")
        po, ldo = _rows(out, n, rows, heads, hd, o, "out")
        need, space = self.attend_workspace(n, rows, heads, max_len), 0
        if need:
            workspace = _space(workspace, need, q, o)
            space, need = workspace.data_ptr(), workspace.numel()
        a = ATTEND_ARGS.pack(
            layer, n, rows, heads, max_len, scale, pq, ldq, po, ldo,
            _whole(lens, (n,), o, i32, "lens"), _whole(counts, (n,), o, i32, "counts"),
            _whole(parents, (n, rows), o, i32, "parents"), space, need)
        _check(self._attend(self.h, a, _stream(o)))
        return out

    def attend_workspace(self, sequences, rows, heads, max_len):
        need = self._workspace(self.h, sequences, rows, heads, max_len)
        if need < 0:
            _check(need)
        return need

    def keep(self, lens, kept, kept_counts):
        """Moves the rows kept [sequences][rows] (ascending row numbers, the first
        kept_counts of each sequence) to positions lens[b], lens[b] + 1, ... in
        every layer. The caller's lengths then grow by kept_counts."""
        o, i32 = self.dev.ordinal, _torch.int32
        n, rows = kept.shape
        _check(lib().q3h_cache_keep(
            self.h, n, rows, _whole(lens, (n,), o, i32, "lens"),
            _whole(kept, (n, rows), o, i32, "kept"),
            _whole(kept_counts, (n,), o, i32, "kept_counts"), _stream(o)))

    def reserve(self, lens, rows, counts=None, ok=None):
        """Pages for positions lens[b] .. lens[b] + counts[b] - 1 (counts None: rows of
        them), own ones: pages of that range that other sequences hold too are copied.
        ok [sequences] (None: not wanted) is set to 1 where a sequence has them, 0 where
        there were too few; returned."""
        o, i32 = self.dev.ordinal, _torch.int32
        n = lens.shape[0]
        _check(self._reserve(
            self.h, n, rows, _whole(lens, (n,), o, i32, "lens"),
            _whole(counts, (n,), o, i32, "counts"), _whole(ok, (n,), o, i32, "ok"), _stream(o)))
        return ok

    def fork(self, sources, lens):
        """Sequence b becomes the first lens[b] positions of what sequence sources[b]
        was (-1: nothing), for all b at once; pages are shared."""
        o, i32 = self.dev.ordinal, _torch.int32
        n = sources.shape[0]
        _check(self._fork(
            self.h, n, _whole(sources, (n,), o, i32, "sources"),
            _whole(lens, (n,), o, i32, "lens"), _stream(o)))

    def release(self, lens):
        """Sequence b keeps the pages of its first lens[b] positions (0: none)."""
        o = self.dev.ordinal
        n = lens.shape[0]
        _check(self._release(
            self.h, n, _whole(lens, (n,), o, _torch.int32, "lens"), _stream(o)))

    def compact(self, used=None):
        """Moves the pages in use to the front; returns their number (used [1], an
        int32 tensor on the device, made when it is None)."""
        o, i32 = self.dev.ordinal, _torch.int32
        if used is None:
            used = _torch.empty(1, dtype=i32, device=self._device)
        _check(self._compact(self.h, _whole(used, (1,), o, i32, "used"), _stream(o)))
        return used

    def copy(self, src, sources, lens):
        """The first lens[b] positions of sequence sources[b] of another cache (-1:
        none) to sequence b, which has the room already."""
        o, i32 = self.dev.ordinal, _torch.int32
        n = sources.shape[0]
        _check(self._copy(
            self.h, src.h, n, _whole(sources, (n,), o, i32, "sources"),
            _whole(lens, (n,), o, i32, "lens"), _stream(o)))

    def page_state(self):
        """(table [sequences][pages of one at most], counts of pages that a sequence
        holds, refs: how many sequences hold a page), int32 copies."""
        if not self.pages:
            _bad("not a cache of pages")
        n, slots = self.table_shape
        table, counts, refs = _torch.empty(
            n * slots + n + self.pages, dtype=_torch.int32, device=self._device).split(
                (n * slots, n, self.pages))
        at = table.data_ptr()
        _check(self._page_state(self.h, at, at + 4 * n * slots, at + 4 * n * (slots + 1),
                                _stream(self.dev.ordinal)))
        return table.view(n, slots), counts, refs

    def destroy(self):
        if self.h:
            _check(self._destroy(self.h))
            self.h = None

    def __del__(self):
        if self.h and self.dev.h:
            self._destroy(self.h)


def _space(workspace, need, like, ordinal):
    """A uint8 tensor of at least need bytes on the device."""
    if workspace is None:
        return _torch.empty(need, dtype=_torch.uint8, device=like.device)
    _ptr(workspace, ordinal, _torch.uint8, "workspace")
    if not workspace.is_contiguous():
        _bad("workspace is not contiguous")
    return workspace


def token_logprobs(dev, logits, tokens, top_k=0, workspace=None):
    """Scores of logits [rows][vocab] (f32 or bf16) at tokens [rows][m] (int32):
    dict of logprobs [rows][m], entropy [rows] and, with top_k, top_ids and
    top_logprobs [rows][top_k] (largest first, of equal ones the lowest token)."""
    torch, L, o = _use_torch(), lib(), dev.ordinal
    f32, i32 = torch.float32, torch.int32
    rows, vocab = logits.shape
    bf16 = logits.dtype is torch.bfloat16
    stride = logits.stride()
    if vocab > 1 and stride[1] != 1:
        _bad("logits: the elements of a row are not side by side")
    at = _ptr(logits, o, torch.bfloat16 if bf16 else f32, "logits")
    m = tokens.shape[1]
    pt = _whole(tokens, (rows, m), o, i32, "tokens")
    need, space = L.q3h_token_logprobs_workspace(rows, vocab, top_k), 0
    if need < 0:
        _check(need)
    if need:
        workspace = _space(workspace, need, logits, o)
        space, need = workspace.data_ptr(), workspace.numel()
    new = logits.new_empty if not bf16 else lambda shape: logits.new_empty(shape, dtype=f32)
    logprobs, entropy = new((rows, m)), new((rows,))
    res = {"logprobs": logprobs, "entropy": entropy}
    ids = top = None
    if top_k > 0:
        res["top_ids"] = ids = tokens.new_empty((rows, top_k))
        res["top_logprobs"] = top = new((rows, top_k))
    a = SCORE_ARGS.pack(
        at, stride[0] if rows > 1 else vocab, BF16 if bf16 else F32, rows, vocab, m, top_k, pt,
        logprobs.data_ptr(), entropy.data_ptr(), ids.data_ptr() if top_k > 0 else 0,
        top.data_ptr() if top_k > 0 else 0, space, need)
    _check(L.q3h_token_logprobs(dev.h, a, _stream(o)))
    return res
