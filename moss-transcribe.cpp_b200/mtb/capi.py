"""ctypes binding of libmoss_transcribe_b200.so (include/mtb_decoder.h).

The Python names mirror the reference's generation interface so callers and
tests read like the reference's own:
  - Decoder.run / prefill / decode_one / logits_from_hidden / rewind / past_len
    -> Qwen3Decoder (src/qwen3_decoder.hpp:37-60)
  - greedy_generate          -> src/generate.cpp:235
  - cpu_speculative_generate -> src/cpu_speculative.cpp:68 (hooks: draft, committed)
  - cpu_ngram_draft / cpu_greedy_choice -> src/cpu_speculative.cpp:27,39
Every call goes to the CUDA library; there is no Python or CPU fallback, and
loading fails loudly when the library or a GPU is missing.

The operators on a caller's own device memory (PagedCache, rope_append,
paged_attention, attention_weights, cache_evict, logits_process) take torch
tensors on the GPU, or anything with the same data_ptr / shape / stride / dtype /
device.
"""
from __future__ import annotations

import ctypes as C
import os
import struct
import sys

import numpy as np

_HERE = os.path.dirname(os.path.abspath(__file__))
# MTB_LIBRARY selects another build of the library (the bounds-check build
# libmoss_transcribe_b200_bc.so, for instance).
LIB_PATH = os.environ.get("MTB_LIBRARY") or os.path.join(os.path.dirname(_HERE), "libmoss_transcribe_b200.so")
_LIB = None

KV_DEFAULT, KV_F32, KV_F16 = -1, 0, 1
STOP_NONE, STOP_EOS, STOP_LIMIT, STOP_ERROR = 0, 1, 2, 3


class SpecParams(C.Structure):
    _fields_ = [("k_max", C.c_int32), ("n_min", C.c_int32), ("n_max", C.c_int32), ("penalty", C.c_float)]


class Counters(C.Structure):
    _fields_ = [("target_calls", C.c_int64), ("drafted_calls", C.c_int64), ("proposed", C.c_int64),
                ("accepted", C.c_int64), ("target_input_tokens", C.c_int64), ("rewinds", C.c_int64),
                ("stop_reason", C.c_int32), ("past_len", C.c_int32)]

    def as_dict(self):
        return {k: getattr(self, k) for k, _ in self._fields_}


DRAFT_FN = C.CFUNCTYPE(C.c_int, C.c_void_p, C.POINTER(C.c_int32), C.c_int, C.c_int, C.POINTER(C.c_int32))
COMMIT_FN = C.CFUNCTYPE(None, C.c_void_p, C.POINTER(C.c_int32), C.c_int, C.c_int, C.c_int)

T_F32, T_F16, T_BF16 = 0, 1, 2
BAD_PAGE, BAD_LEN, BAD_TOKENS, BAD_WAIT = 1, 2, 4, 8
ROPE_PLAIN, ROPE_LINEAR, ROPE_NTK, ROPE_YARN, ROPE_BANDS = range(5)
ATTENTION_WORKSPACE = 64 << 20
PAGE = 64


class PagedCacheView(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("type", C.c_int32), ("head_dim", C.c_int32),
                ("n_kv_heads", C.c_int32), ("n_pages", C.c_int32), ("page_stride", C.c_int64), ("head_stride", C.c_int64),
                ("page_table", C.c_void_p), ("table_stride", C.c_int32), ("n_seq", C.c_int32), ("kv_len", C.c_void_p),
                ("position", C.c_void_p), ("weight", C.c_void_p), ("status", C.c_void_p)]


class LogitsParams(C.Structure):
    _fields_ = [("history", C.c_void_p), ("history_len", C.c_int64), ("history_begin", C.c_void_p), ("history_end", C.c_void_p),
                ("repetition", C.c_void_p), ("presence", C.c_void_p), ("frequency", C.c_void_p), ("bias_ids", C.c_void_p),
                ("bias_values", C.c_void_p), ("bias_len", C.c_int64), ("bias_begin", C.c_void_p), ("bias_end", C.c_void_p), ("mask", C.c_void_p),
                ("mask_stride", C.c_int64), ("mask_rows", C.c_int32), ("mask_row", C.c_void_p)]


# Every exported function with (restype, argtypes); used for binding and for
# the export check of the boundary test.
_vp, _i32p, _f32p, _ip = C.c_void_p, C.POINTER(C.c_int32), C.POINTER(C.c_float), C.POINTER(C.c_int)
SIGNATURES = {
    "moss_transcribe_capi_abi_version": (C.c_int, []),
    "moss_transcribe_capi_load": (_vp, [C.c_char_p]),
    "moss_transcribe_capi_free": (None, [_vp]),
    "moss_transcribe_capi_transcribe_path": (_vp, [_vp, C.c_char_p, C.c_int]),
    "moss_transcribe_capi_transcribe_pcm": (_vp, [_vp, _f32p, C.c_int, C.c_int, C.c_int]),
    "moss_transcribe_capi_free_string": (None, [_vp]),
    "moss_transcribe_capi_last_error": (C.c_char_p, [_vp]),
    "mtb_abi_version": (C.c_int, []),
    "mtb_global_error": (C.c_char_p, []),
    "mtb_model_load": (C.c_int, [C.c_char_p, C.c_int, C.POINTER(_vp)]),
    "mtb_model_free": (None, [_vp]),
    "mtb_model_error": (C.c_char_p, [_vp]),
    "mtb_model_dims": (C.c_int, [_vp, _i32p]),
    "mtb_model_persistent_grid": (C.c_int, [_vp]),
    "mtb_decoder_create": (C.c_int, [_vp, C.c_int, C.c_int, C.c_int, C.POINTER(_vp)]),
    "mtb_decoder_free": (None, [_vp]),
    "mtb_decoder_error": (C.c_char_p, [_vp]),
    "mtb_decoder_past_len": (C.c_int, [_vp]),
    "mtb_decoder_reset": (C.c_int, [_vp]),
    "mtb_decoder_rewind": (C.c_int, [_vp, C.c_int]),
    "mtb_decoder_run": (C.c_int, [_vp, _f32p, C.c_int, _f32p]),
    "mtb_decoder_logits": (C.c_int, [_vp, _f32p, _f32p]),
    "mtb_decoder_kv_read": (C.c_int, [_vp, C.c_int, C.c_int, C.c_int, C.c_int, _f32p]),
    "mtb_decoder_fill_synthetic_kv": (C.c_int, [_vp, C.c_int, C.c_uint32]),
    "mtb_greedy_generate": (C.c_int, [_vp, _f32p, C.c_int, C.c_int, C.c_int, C.c_float, _i32p, _ip]),
    "mtb_spec_generate": (C.c_int, [_vp, _f32p, C.c_int, C.c_int, C.c_int, C.POINTER(SpecParams), _i32p, _ip,
                                    C.POINTER(Counters), DRAFT_FN, COMMIT_FN, _vp]),
    "mtb_fuse_embeds": (C.c_int, [_vp, _i32p, C.c_int, _f32p, C.c_int, C.c_int, _f32p]),
    "mtb_spec_generate_ids": (C.c_int, [_vp, _i32p, C.c_int, _f32p, C.c_int, C.c_int, C.c_int, C.c_int,
                                        C.POINTER(SpecParams), _i32p, _ip, C.POINTER(Counters)]),
    "mtb_resume": (C.c_int, [_vp, _i32p, C.c_int, C.c_int, C.c_int, C.c_int, C.POINTER(SpecParams)]),
    "mtb_spec_step": (C.c_int, [_vp, _i32p, C.c_int, C.POINTER(Counters)]),
    "mtb_spec_step_async": (C.c_int, [_vp, _vp, C.c_int]),
    "mtb_spec_prime": (C.c_int, [_vp, _f32p, C.c_int, C.c_int, C.c_int, C.POINTER(SpecParams)]),
    "mtb_spec_step_group_async": (C.c_int, [C.POINTER(_vp), C.c_int]),
    "mtb_spec_run_group": (C.c_int, [C.POINTER(_vp), C.c_int, C.c_int, _ip]),
    "mtb_snapshot_save": (C.c_int, [_vp]),
    "mtb_snapshot_restore_async": (C.c_int, [_vp]),
    "mtb_read_ids": (C.c_int, [_vp, _i32p, C.c_int, _ip, C.POINTER(Counters)]),
    "mtb_sync": (C.c_int, [_vp]),
    "mtb_event_record": (C.c_int, [_vp, C.c_int]),
    "mtb_event_elapsed_ms": (C.c_int, [_vp, C.c_int, C.c_int, _f32p]),
    "mtb_step_kernel_launches": (C.c_int, [_vp]),
    "mtb_transfer_bytes": (C.c_int, [_vp, C.POINTER(C.c_int64), C.POINTER(C.c_int64)]),
    "mtb_step_timeline": (C.c_int, [_vp, C.POINTER(C.c_int64), C.c_int, _ip]),
    "mtb_step_capture": (C.c_int, [_vp, _vp, _vp, _vp, _vp, _ip]),
    "mtb_capi_can_transcribe": (C.c_int, []),
    "mtb_set_log_level": (None, [C.c_int]),
    "mtb_spec_params_from_env": (C.c_int, [C.POINTER(SpecParams)]),
    "mtb_kv_type_from_env": (C.c_int, []),
    "mtb_debug_fail_alloc": (None, [C.c_int]),
    "mtb_f16_slices_per_block": (C.c_int, [C.c_int, C.c_int]),
    "mtb_bounds_check_enabled": (C.c_int, []),
    "mtb_bounds_check_status": (C.c_int, [C.c_int]),
    "mtb_format_generation_log": (C.c_int, [_vp, C.c_int, C.c_int, _vp, C.c_int, C.c_double, C.c_double, C.c_int,
                                            C.c_char_p, C.c_int]),
    "mtb_debug_poison_kv": (C.c_int, [_vp, C.c_int, C.c_int]),
    "mtb_ngram_draft": (C.c_int, [_vp, _i32p, C.c_int, C.c_int, C.c_int, C.c_int, _i32p, _ip]),
    "mtb_greedy_choice": (C.c_int, [_vp, _f32p, C.c_int, _i32p, C.c_int, C.c_float, _i32p]),
    "mtb_lm_head_argmax_noalloc": (C.c_int, [_vp, _vp, C.c_int, _vp, _vp]),
    "mtb_noalloc_error": (C.c_char_p, []),
    "mtb_audio_load": (C.c_int, [C.c_char_p, C.c_int, C.POINTER(_vp)]),
    "mtb_audio_free": (None, [_vp]),
    "mtb_audio_error": (C.c_char_p, [_vp]),
    "mtb_audio_dims": (C.c_int, [_vp, _i32p]),
    "mtb_audio_tokens": (C.c_int, [_vp, C.c_int]),
    "mtb_audio_encode": (C.c_int, [_vp, _f32p, C.c_int, _f32p, C.c_int, _ip]),
    "mtb_audio_last_ms": (C.c_float, [_vp]),
    "mtb_audio_debug_chunk": (C.c_int, [_vp, _f32p, C.c_int, _f32p, _f32p]),
    "mtb_rope_frequencies": (C.c_int, [C.c_int, C.c_double, C.c_int, C.c_double, C.c_double, C.c_double, C.c_double,
                                       C.POINTER(C.c_double), _f32p]),
    "mtb_rope_append": (C.c_int, [_vp, _vp, C.c_int, _vp, C.c_int, _vp, C.c_int64, C.c_int, _vp, C.c_int64, _vp,
                                  C.c_int64, _vp, C.c_int, C.c_int, C.c_float, _vp, C.c_int64, _vp]),
    "mtb_paged_attention": (C.c_int, [_vp, _vp, C.c_int, C.c_int, _vp, C.c_int64, C.c_int, C.c_float, _vp, C.c_int64,
                                      _vp, _vp, C.c_size_t, _vp]),
    "mtb_attention_weights": (C.c_int, [_vp, _vp, C.c_int, C.c_int, _vp, C.c_int64, C.c_int, C.c_float, _vp, C.c_float,
                                        _vp]),
    "mtb_debug_stall_attention": (None, [C.c_int]),
    "mtb_cache_evict_workspace": (C.c_int64, [C.c_int, C.c_int, C.c_int]),
    "mtb_cache_evict": (C.c_int, [_vp, C.c_int, C.c_int, C.c_int, _vp, _vp, C.c_size_t, _vp]),
    "mtb_logits_process": (C.c_int, [_vp, C.c_int, C.c_int, C.c_int, C.c_int64, _vp, _vp, C.c_int64, _vp, _vp]),
}


class MtbError(RuntimeError):
    pass


def lib():
    """The loaded CUDA library; raises if it has not been built."""
    global _LIB
    if _LIB is None:
        if not os.path.exists(LIB_PATH):
            raise MtbError(f"{LIB_PATH} is missing: build it with __graft_entry__.build() or `make -C "
                           f"{os.path.dirname(LIB_PATH)}`")
        L = C.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(L, name)
            fn.restype = res
            fn.argtypes = args
        _LIB = L
    return _LIB


def spec_params_from_env() -> dict:
    """The policy a NULL params pointer selects: the reference policy (k 4,
    n-grams 16..2, penalty from MTD_REPETITION_PENALTY) with MTB_SPEC_K /
    MTB_NGRAM_MIN / MTB_NGRAM_MAX overrides.  Raises on an invalid variable."""
    p = SpecParams()
    if lib().mtb_spec_params_from_env(C.byref(p)) != 0:
        raise MtbError(lib().mtb_global_error().decode())
    return {"k_max": p.k_max, "n_min": p.n_min, "n_max": p.n_max, "penalty": p.penalty}


def kv_type_from_env() -> int:
    """KV_F32 or KV_F16 as MTB_KV_DTYPE selects (unset: KV_F32); -1 if unknown."""
    return lib().mtb_kv_type_from_env()


def debug_fail_alloc(n: int) -> None:
    """Test hook: the n-th device allocation from now on fails (0: off)."""
    lib().mtb_debug_fail_alloc(int(n))


def _f32(a):
    return a.ctypes.data_as(_f32p)


def _i32(a):
    return a.ctypes.data_as(_i32p)


def _arr_i32(x):
    return np.ascontiguousarray(np.asarray(x, dtype=np.int32))


class Model:
    """Decoder weights of a GGUF file resident on one CUDA device."""

    def __init__(self, gguf_path: str, device: int = 0):
        L = lib()
        p = C.c_void_p()
        rc = L.mtb_model_load(gguf_path.encode(), int(device), C.byref(p))
        if rc != 0:
            raise MtbError(f"mtb_model_load: {L.mtb_global_error().decode()}")
        self.ptr = p
        self.device = device
        dims = (C.c_int32 * 8)()
        L.mtb_model_dims(self.ptr, dims)
        (self.hidden, self.n_layers, self.n_heads, self.n_kv_heads, self.head_dim, self.ffn, self.vocab,
         self.eos) = list(dims)
        self.persistent_grid = L.mtb_model_persistent_grid(self.ptr)

    def close(self):
        if getattr(self, "ptr", None):
            lib().mtb_model_free(self.ptr)
            self.ptr = None

    def __del__(self):
        self.close()


class AudioEncoder:
    """The audio front end of a GGUF on one CUDA device: mt::AudioEncoder
    (src/audio_encoder.hpp:23-34), encode(samples16k) -> rows [n_tokens][hidden]."""

    def __init__(self, gguf_path: str, device: int = 0):
        L = lib()
        p = C.c_void_p()
        if L.mtb_audio_load(gguf_path.encode(), int(device), C.byref(p)) != 0:
            raise MtbError(f"mtb_audio_load: {L.mtb_audio_error(None).decode()}")
        self.ptr = p
        dims = (C.c_int32 * 10)()
        L.mtb_audio_dims(self.ptr, dims)
        (self.hidden, self.d_model, self.n_layers, self.n_heads, self.ffn, self.n_mels, self.n_frames,
         self.chunk_samples, self.enc_frames, self.merge) = list(dims)

    def close(self):
        if getattr(self, "ptr", None):
            lib().mtb_audio_free(self.ptr)
            self.ptr = None

    def __del__(self):
        self.close()

    def _check(self, rc, what):
        if rc != 0:
            raise MtbError(f"{what}: {lib().mtb_audio_error(self.ptr).decode()}")

    def tokens(self, n_samples: int) -> int:
        return lib().mtb_audio_tokens(self.ptr, int(n_samples))

    def encode(self, samples16k: np.ndarray, max_tokens: int | None = None) -> np.ndarray:
        x = np.ascontiguousarray(samples16k, dtype=np.float32)
        cap = max(self.tokens(len(x)), 1) if max_tokens is None else max_tokens
        out = np.zeros((max(cap, 1), self.hidden), dtype=np.float32)
        n = C.c_int(0)
        self._check(lib().mtb_audio_encode(self.ptr, _f32(x), int(len(x)), _f32(out), int(cap), C.byref(n)),
                    "mtb_audio_encode")
        return out[:n.value]

    def last_ms(self) -> float:
        return float(lib().mtb_audio_last_ms(self.ptr))

    def debug_chunk(self, chunk: np.ndarray):
        """(mel [n_mels][frames], encoder output [enc_frames][d_model]) of one chunk."""
        x = np.ascontiguousarray(chunk, dtype=np.float32)
        mel = np.zeros((self.n_mels, self.n_frames), dtype=np.float32)
        enc = np.zeros((self.enc_frames, self.d_model), dtype=np.float32)
        self._check(lib().mtb_audio_debug_chunk(self.ptr, _f32(x), int(len(x)), _f32(mel), _f32(enc)),
                    "mtb_audio_debug_chunk")
        return mel, enc


class Decoder:
    """Qwen3Decoder on the GPU: paged KV cache plus the device step state."""

    def __init__(self, model: Model, max_seq: int, kv_type: int = KV_F32, max_new: int = 4096):
        L = lib()
        p = C.c_void_p()
        if L.mtb_decoder_create(model.ptr, int(max_seq), int(kv_type), int(max_new), C.byref(p)) != 0:
            raise MtbError(f"mtb_decoder_create: {L.mtb_global_error().decode()}")
        self.ptr = p
        self.model = model
        self.max_seq = max_seq
        self.max_new = max_new

    def close(self):
        if getattr(self, "ptr", None):
            lib().mtb_decoder_free(self.ptr)
            self.ptr = None

    def __del__(self):
        self.close()

    def _check(self, rc, what):
        if rc != 0:
            raise MtbError(f"{what}: {lib().mtb_decoder_error(self.ptr).decode()}")

    # -- Qwen3Decoder surface ------------------------------------------------
    @property
    def past_len(self) -> int:
        v = lib().mtb_decoder_past_len(self.ptr)
        if v < 0:
            self._check(-1, "past_len")
        return v

    def reset(self):
        self._check(lib().mtb_decoder_reset(self.ptr), "reset")

    def rewind(self, position: int) -> bool:
        return lib().mtb_decoder_rewind(self.ptr, int(position)) == 0

    def run(self, embeds: np.ndarray) -> np.ndarray:
        e = np.ascontiguousarray(embeds, dtype=np.float32).reshape(-1, self.model.hidden)
        out = np.zeros_like(e)
        self._check(lib().mtb_decoder_run(self.ptr, _f32(e), e.shape[0], _f32(out)), "run")
        return out

    def prefill(self, embeds: np.ndarray) -> np.ndarray:
        self.reset()
        return self.run(embeds)

    def decode_one(self, embed: np.ndarray) -> np.ndarray:
        return self.run(np.asarray(embed, dtype=np.float32).reshape(1, -1))[0]

    def logits_from_hidden(self, hidden_row: np.ndarray) -> np.ndarray:
        h = np.ascontiguousarray(hidden_row, dtype=np.float32).ravel()
        out = np.zeros(self.model.vocab, dtype=np.float32)
        self._check(lib().mtb_decoder_logits(self.ptr, _f32(h), _f32(out)), "logits")
        return out

    def kv(self, layer: int, which: int, pos0: int, n: int) -> np.ndarray:
        out = np.zeros((n, self.model.n_kv_heads, self.model.head_dim), dtype=np.float32)
        self._check(lib().mtb_decoder_kv_read(self.ptr, layer, which, pos0, n, _f32(out)), "kv_read")
        return out

    def fill_synthetic_kv(self, n_pos: int, seed: int):
        self._check(lib().mtb_decoder_fill_synthetic_kv(self.ptr, int(n_pos), int(seed) & 0xFFFFFFFF), "fill_kv")

    # -- generation ------------------------------------------------------------
    def greedy_generate(self, fused: np.ndarray, max_new: int, eos: int, penalty: float = 1.0) -> list[int]:
        f = np.ascontiguousarray(fused, dtype=np.float32).reshape(-1, self.model.hidden)
        out = np.zeros(max_new, dtype=np.int32)
        n = C.c_int()
        self._check(lib().mtb_greedy_generate(self.ptr, _f32(f), f.shape[0], int(max_new), int(eos), float(penalty),
                                              _i32(out), C.byref(n)), "greedy_generate")
        return out[:n.value].tolist()

    def cpu_speculative_generate(self, fused: np.ndarray, max_new: int, eos: int, k_max: int = 4, n_min: int = 2,
                                 n_max: int = 16, penalty: float = 1.0, draft=None, committed=None,
                                 reference_policy: bool = False):
        """Strict speculative generate; `draft(ids, budget)` and
        `committed(ids, past_len, stopped)` are the reference's hooks.
        reference_policy: pass no parameters (k 4, n 16..2, the penalty from
        MTD_REPETITION_PENALTY), as the reference's own call does."""
        f = np.ascontiguousarray(fused, dtype=np.float32).reshape(-1, self.model.hidden)
        out = np.zeros(max_new, dtype=np.int32)
        n = C.c_int()
        counters = Counters()
        params = SpecParams(k_max, n_min, n_max, penalty)

        def _draft(user, ids, n_ids, budget, dst):
            got = list(draft([ids[i] for i in range(n_ids)], budget))[:budget]
            for i, v in enumerate(got):
                dst[i] = int(v)
            return len(got)

        def _commit(user, ids, n_ids, past, stopped):
            committed([ids[i] for i in range(n_ids)], past, bool(stopped))

        dfn = DRAFT_FN(_draft) if draft else DRAFT_FN()
        cfn = COMMIT_FN(_commit) if committed else COMMIT_FN()
        self._check(lib().mtb_spec_generate(self.ptr, _f32(f), f.shape[0], int(max_new), int(eos),
                                            None if reference_policy else C.byref(params),
                                            _i32(out), C.byref(n), C.byref(counters), dfn, cfn, None),
                    "spec_generate")
        return out[:n.value].tolist(), counters.as_dict()

    # -- step-level API --------------------------------------------------------
    def fuse_embeds(self, ids, audio: np.ndarray, audio_token_id: int) -> np.ndarray:
        """fuse_embeds (src/generate.cpp:113) with the rows built on the device."""
        a = _arr_i32(ids)
        au = np.ascontiguousarray(audio, dtype=np.float32).reshape(-1, self.model.hidden)
        out = np.zeros((a.size, self.model.hidden), dtype=np.float32)
        self._check(lib().mtb_fuse_embeds(self.ptr, _i32(a), a.size, _f32(au), au.shape[0], int(audio_token_id),
                                          _f32(out)), "fuse_embeds")
        return out

    def spec_generate_ids(self, ids, audio: np.ndarray, audio_token_id: int, max_new: int, eos: int, k_max: int = 4,
                          n_min: int = 2, n_max: int = 16, penalty: float = 1.0):
        """Strict speculative generate from ids + audio rows, fused on the device."""
        a = _arr_i32(ids)
        au = np.ascontiguousarray(audio, dtype=np.float32).reshape(-1, self.model.hidden)
        out = np.zeros(max_new, dtype=np.int32)
        n = C.c_int()
        counters = Counters()
        params = SpecParams(k_max, n_min, n_max, penalty)
        self._check(lib().mtb_spec_generate_ids(self.ptr, _i32(a), a.size, _f32(au), au.shape[0], int(audio_token_id),
                                                int(max_new), int(eos), C.byref(params), _i32(out), C.byref(n),
                                                C.byref(counters)), "spec_generate_ids")
        return out[:n.value].tolist(), counters.as_dict()

    def resume(self, ids, past: int, max_new: int, eos: int, k_max=4, n_min=2, n_max=16, penalty=1.0):
        a = _arr_i32(ids)
        params = SpecParams(k_max, n_min, n_max, penalty)
        self._check(lib().mtb_resume(self.ptr, _i32(a), a.size, int(past), int(max_new), int(eos), C.byref(params)),
                    "resume")

    def spec_step(self, draft=None) -> dict:
        c = Counters()
        if draft is None:
            rc = lib().mtb_spec_step(self.ptr, None, 0, C.byref(c))
        else:
            a = _arr_i32(draft)
            rc = lib().mtb_spec_step(self.ptr, _i32(a) if a.size else _i32(np.zeros(1, np.int32)), a.size, C.byref(c))
        self._check(rc, "spec_step")
        return c.as_dict()

    def read_ids(self):
        out = np.zeros(self.max_new, dtype=np.int32)
        n = C.c_int()
        c = Counters()
        self._check(lib().mtb_read_ids(self.ptr, _i32(out), self.max_new, C.byref(n), C.byref(c)), "read_ids")
        return out[:n.value].tolist(), c.as_dict()

    def cpu_ngram_draft(self, history, maximum: int, n_min: int = 2, n_max: int = 16) -> list[int]:
        h = _arr_i32(history)
        out = np.zeros(max(1, len(h) + 16), dtype=np.int32)
        n = C.c_int()
        self._check(lib().mtb_ngram_draft(self.ptr, _i32(h) if h.size else None, h.size, int(maximum), int(n_min),
                                          int(n_max), _i32(out), C.byref(n)), "ngram_draft")
        return out[:n.value].tolist()

    def cpu_greedy_choice(self, raw, history, penalty: float) -> int:
        r = np.ascontiguousarray(np.asarray(raw, dtype=np.float32))
        h = _arr_i32(history)
        c = C.c_int32()
        self._check(lib().mtb_greedy_choice(self.ptr, _f32(r), r.size, _i32(h) if h.size else None, h.size,
                                            float(penalty), C.byref(c)), "greedy_choice")
        return c.value

    # -- timing ----------------------------------------------------------------
    def sync(self):
        self._check(lib().mtb_sync(self.ptr), "sync")

    def step_kernel_launches(self) -> int:
        return lib().mtb_step_kernel_launches(self.ptr)

    def step_timeline(self):
        """(arrive_ns, release_ns) per grid barrier and (start, end) of the last
        persistent step; needs MTB_PROFILE=1 when the decoder was created."""
        out = (C.c_int64 * (6 * 512 + 2 + 256 * 512 * 17))()
        n = C.c_int()
        self._check(lib().mtb_step_timeline(self.ptr, out, len(out), C.byref(n)), "step_timeline")
        vals = np.frombuffer(out, dtype=np.int64)
        marks = [tuple(vals[1026 + 4 * b:1030 + 4 * b]) for b in range(512)]
        self.last_arrivals = vals[6 * 512 + 2:6 * 512 + 2 + 256 * 512].reshape(256, 512)
        self.last_cta_marks = vals[6 * 512 + 2 + 256 * 512:].reshape(256, 512, 16)
        return [(vals[2 * b], vals[2 * b + 1]) for b in range(512)], (vals[1024], vals[1025]), marks

    def step_capture(self):
        """The last persistent step's own outputs (MTB_STEP_CAPTURE=1 when the
        decoder was created): final-normed rows [T][hidden], LM-head maxima
        [T], their first indices [T] and the per-stream (rows, first row)."""
        hid = np.zeros((16, self.model.hidden), dtype=np.float32)
        mv = np.zeros(16, dtype=np.float32)
        mi = np.zeros(16, dtype=np.int32)
        sr = np.zeros((8, 2), dtype=np.int32)
        n = C.c_int()
        self._check(lib().mtb_step_capture(self.ptr, hid.ctypes.data, mv.ctypes.data, mi.ctypes.data, sr.ctypes.data,
                                           C.byref(n)), "step_capture")
        T = n.value
        return hid[:T], mv[:T], mi[:T], sr

    def poison_kv(self, pos0: int, n_pos: int):
        """Test hook: NaN into cache positions [pos0, pos0 + n_pos) of every layer."""
        self._check(lib().mtb_debug_poison_kv(self.ptr, int(pos0), int(n_pos)), "poison_kv")

    def transfer_bytes(self):
        a, b = C.c_int64(), C.c_int64()
        lib().mtb_transfer_bytes(self.ptr, C.byref(a), C.byref(b))
        return a.value, b.value

    def spec_prime(self, fused: np.ndarray, max_new: int, eos: int, k_max: int = 4, n_min: int = 2, n_max: int = 16,
                   penalty: float = 1.0):
        """Parameters + prefill of the fused rows (first id emitted), no decoding."""
        f = np.ascontiguousarray(fused, dtype=np.float32).reshape(-1, self.model.hidden)
        params = SpecParams(k_max, n_min, n_max, penalty)
        self._check(lib().mtb_spec_prime(self.ptr, _f32(f), f.shape[0], int(max_new), int(eos), C.byref(params)),
                    "spec_prime")

    def spec_step_async(self, draft_device_ptr, n_draft: int):
        self._check(lib().mtb_spec_step_async(self.ptr, C.c_void_p(draft_device_ptr), int(n_draft)), "spec_step_async")

    def snapshot_save(self):
        self._check(lib().mtb_snapshot_save(self.ptr), "snapshot_save")

    def snapshot_restore_async(self):
        self._check(lib().mtb_snapshot_restore_async(self.ptr), "snapshot_restore")

    def event_record(self, slot: int):
        self._check(lib().mtb_event_record(self.ptr, int(slot)), "event_record")

    def event_elapsed_ms(self, a: int, b: int) -> float:
        ms = C.c_float()
        self._check(lib().mtb_event_elapsed_ms(self.ptr, int(a), int(b), C.byref(ms)), "event_elapsed")
        return ms.value


def format_generation_log(ids, eos: int, counters: dict, k_max: int, prefill_s: float = 0.0,
                          decoder_s: float = 0.0, trace: bool = True) -> str:
    """The reference's end-of-generation lines for given results (no GPU needed)."""
    a = _arr_i32(ids)
    c = Counters(*(int(counters[k]) for k in ("target_calls", "drafted_calls", "proposed", "accepted",
                                                 "target_input_tokens", "rewinds", "stop_reason", "past_len")))
    n = lib().mtb_format_generation_log(_i32(a) if a.size else None, a.size, int(eos), C.byref(c), int(k_max),
                                        float(prefill_s), float(decoder_s), int(trace), None, 0)
    buf = C.create_string_buffer(n + 1)
    lib().mtb_format_generation_log(_i32(a) if a.size else None, a.size, int(eos), C.byref(c), int(k_max),
                                    float(prefill_s), float(decoder_s), int(trace), buf, n + 1)
    return buf.value.decode()


def _group(decoders):
    arr = (_vp * len(decoders))(*[d.ptr for d in decoders])
    return arr


def _group_error(decoders, what):
    msg = lib().mtb_decoder_error(decoders[0].ptr).decode() if decoders else ""
    return MtbError(f"{what}: {msg or lib().mtb_global_error().decode()}")


def spec_step_group_async(decoders):
    """One verify step of several decoders of one model as one launch (mtb_spec_step_group_async)."""
    if lib().mtb_spec_step_group_async(_group(decoders), len(decoders)) != 0:
        raise _group_error(decoders, "spec_step_group_async")


def spec_run_group(decoders, max_steps: int = 0) -> int:
    """Group steps until every decoder stopped; returns the steps launched (mtb_spec_run_group)."""
    n = C.c_int()
    if lib().mtb_spec_run_group(_group(decoders), len(decoders), int(max_steps), C.byref(n)) != 0:
        raise _group_error(decoders, "spec_run_group")
    return n.value


# ---- operators on a caller's own device memory -----------------------------
# A step's calls take a few microseconds on the device, so what is done here for each call is kept short.


class _Names(dict):
    """dtype object -> its name, filled as dtypes are met."""

    def __missing__(self, dtype):
        name = self[dtype] = str(dtype).rsplit(".", 1)[-1]
        return name


_NAME = _Names()
_CODES = {"float32": T_F32, "float16": T_F16, "bfloat16": T_BF16}
_PACK_CACHE = struct.Struct("@PPiiiiqqPiiPPPP").pack  # mtb_paged_cache
_PACK_LOGITS = struct.Struct("@PqPPPPPPPqPPPqiP").pack  # mtb_logits_params
assert struct.calcsize("@PPiiiiqqPiiPPPP") == C.sizeof(PagedCacheView)
assert struct.calcsize("@PqPPPPPPPqPPPqiP") == C.sizeof(LogitsParams)


def _need(ok, what):
    if not ok:
        raise MtbError(what)


def _shape(t, name, dims):
    shape = t.shape
    if len(shape) != dims:
        raise MtbError(f"{name} must have {dims} dimensions")
    return shape


def _flat(t, name, dtype, n, device):
    """The pointer of a tensor without gaps on `device`, 0 for None; n: the least number of its elements."""
    if t is None:
        return 0
    if _NAME[t.dtype] != dtype or not t.is_contiguous() or t.numel() < n or t.get_device() != device:
        raise MtbError(f"{name} must be contiguous {dtype} with at least {n} elements on the others' device")
    return t.data_ptr()


def _rows(t, name, tokens, heads, dim, dtype, device):
    """(pointer, elements between tokens) of [tokens][heads][dim] whose tokens' rows have no gaps."""
    if t.shape == (tokens, heads, dim) and _NAME[t.dtype] == dtype and t.get_device() == device:
        s0, s1, s2 = t.stride()
        if s2 == 1 and (s1 == dim or heads == 1):
            return t.data_ptr(), (s0 if tokens > 1 else max(s0, heads * dim))
    raise MtbError(f"{name} must be {dtype} [{tokens}][{heads}][{dim}] on the cache's device with a token's rows contiguous")


def _space(t, device):
    """(pointer, bytes) of a workspace."""
    if not t.is_contiguous() or t.get_device() != device:
        raise MtbError("workspace must be contiguous, on the cache's device")
    return t.data_ptr(), t.numel() * t.element_size()


def _stream(device, stream):
    """A cudaStream_t: the one given, else torch's current stream of the device."""
    if stream is not None:
        return stream if isinstance(stream, int) else stream.cuda_stream
    torch = sys.modules.get("torch")
    return torch._C._cuda_getCurrentRawStream(device) if torch is not None and device >= 0 else 0


def _ok(rc, what):
    if rc != 0:
        raise MtbError(f"{what}: {lib().mtb_global_error().decode()}")


class PagedCache:
    """A view of one layer's paged cache (mtb_paged_cache): k and v [pages][kv_heads][64][head_dim] with equal strides
    (their pages and heads may be apart, as in one layer of a larger pool), page_table [sequences][pages of one], kv_len
    [sequences] with the new tokens included; position (int32) and weight (f32) [pages][kv_heads][64] and status (int32,
    BAD_* bits) where wanted.  It keeps the tensors alive and may be used for any number of calls."""

    __slots__ = ("kept", "heads", "dim", "type", "n_seq", "table_len", "device", "view")

    def __init__(self, k, v, page_table, kv_len, position=None, weight=None, status=None):
        shape, strides, name, device = k.shape, k.stride(), _NAME[k.dtype], k.get_device()
        if len(shape) != 4 or shape[2] != PAGE or strides[3] != 1 or strides[2] != shape[3]:
            raise MtbError("k must be [pages][kv_heads][64][head_dim] with a page's rows contiguous")
        if v.shape != shape or v.stride() != strides or v.dtype != k.dtype or v.get_device() != device:
            raise MtbError("v must have k's shape, strides, type and device")
        if name != "float16" and name != "bfloat16":
            raise MtbError("the cache's type is float16 or bfloat16")
        pages, heads, _, dim = shape
        n_seq, table_len = _shape(page_table, "page_table", 2)
        meta, block = pages * heads * PAGE, PAGE * dim
        self.kept = (k, v, page_table, kv_len, position, weight, status)
        self.heads, self.dim, self.type, self.n_seq, self.table_len, self.device = heads, dim, name, n_seq, table_len, device
        self.view = _PACK_CACHE(
            k.data_ptr(), v.data_ptr(), _CODES[name], dim, heads, pages, strides[0] if pages > 1 else max(strides[0], heads * block),
            strides[1] if heads > 1 else max(strides[1], block), _flat(page_table, "page_table", "int32", 0, device), table_len, n_seq,
            _flat(kv_len, "kv_len", "int32", n_seq, device), _flat(position, "position", "int32", meta, device),
            _flat(weight, "weight", "float32", meta, device), _flat(status, "status", "int32", 1, device))


def rope_frequencies(rotary_dim: int, base: float, kind: int = ROPE_PLAIN, factor: float = 1.0, original_len: float = 0.0,
                     fast: float = 32.0, slow: float = 1.0):
    """(inverse frequencies float64 [rotary_dim / 2], scale of cos and sin) for rope_append; needs no GPU."""
    out = np.zeros(max(rotary_dim // 2, 0), dtype=np.float64)
    scale = C.c_float()
    _ok(lib().mtb_rope_frequencies(int(rotary_dim), float(base), int(kind), float(factor), float(original_len), float(fast),
                                   float(slow), out.ctypes.data_as(C.POINTER(C.c_double)), C.byref(scale)), "rope_frequencies")
    return out, scale.value


def rope_append(cache: PagedCache, cu_tokens, positions, q, k, v, inv_freq, q_out, interleaved: bool = False,
                factor: float = 1.0, stream=None):
    """Rotary positions of q and k and the append of k and v to the cache (mtb_rope_append).  q [tokens][heads][dim], k and v
    [tokens][kv_heads][dim] (views of a fused projection's rows will do), inv_freq float64 [rotary / 2], q_out of the
    cache's type.  Token i of a sequence's n goes to slot kv_len - n + i."""
    n, heads, _ = _shape(q, "q", 3)
    name, dim, dev = _NAME[q.dtype], cache.dim, cache.device
    qp, qs = _rows(q, "q", n, heads, dim, name, dev)
    kp, ks = _rows(k, "k", n, cache.heads, dim, name, dev)
    vp, vs = _rows(v, "v", n, cache.heads, dim, name, dev)
    op, os_ = _rows(q_out, "q_out", n, heads, dim, cache.type, dev)
    rc = lib().mtb_rope_append(cache.view, _flat(cu_tokens, "cu_tokens", "int32", cache.n_seq + 1, dev), n,
                               _flat(positions, "positions", "int32", n, dev), _CODES.get(name, -1), qp, qs, heads, kp, ks, vp, vs,
                               _flat(inv_freq, "inv_freq", "float64", 0, dev), 2 * inv_freq.numel(), interleaved, factor, op, os_,
                               _stream(dev, stream))
    if rc != 0:
        _ok(rc, "rope_append")


def paged_attention(cache: PagedCache, cu_tokens, q, out, workspace, lse=None, scale: float | None = None, max_tokens: int = 0,
                    stream=None):
    """Causal attention of the new tokens over the cache (mtb_paged_attention).  q and out [tokens][heads][dim] of the
    cache's type, lse f32 [tokens][heads]; workspace: ATTENTION_WORKSPACE bytes, zeroed once before its first use and not
    shared by calls that overlap."""
    n, heads, _ = _shape(q, "q", 3)
    dim, dev = cache.dim, cache.device
    qp, qs = _rows(q, "q", n, heads, dim, cache.type, dev)
    op, os_ = _rows(out, "out", n, heads, dim, cache.type, dev)
    wp, wn = _space(workspace, dev)
    rc = lib().mtb_paged_attention(cache.view, _flat(cu_tokens, "cu_tokens", "int32", cache.n_seq + 1, dev), n, max_tokens, qp, qs, heads,
                                   dim ** -0.5 if scale is None else scale, op, os_, _flat(lse, "lse", "float32", n * heads, dev), wp, wn,
                                   _stream(dev, stream))
    if rc != 0:
        _ok(rc, "paged_attention")


def attention_weights(cache: PagedCache, cu_tokens, q, lse, decay: float = 1.0, scale: float | None = None, max_tokens: int = 0,
                      stream=None):
    """cache weight = decay * weight + the softmax weight each position received in that attention (mtb_attention_weights)."""
    n, heads, _ = _shape(q, "q", 3)
    dim, dev = cache.dim, cache.device
    qp, qs = _rows(q, "q", n, heads, dim, cache.type, dev)
    rc = lib().mtb_attention_weights(cache.view, _flat(cu_tokens, "cu_tokens", "int32", cache.n_seq + 1, dev), n, max_tokens, qp, qs, heads,
                                     dim ** -0.5 if scale is None else scale, _flat(lse, "lse", "float32", n * heads, dev), decay,
                                     _stream(dev, stream))
    if rc != 0:
        _ok(rc, "attention_weights")


def cache_evict_workspace(n_seq: int, n_kv_heads: int, table_stride: int) -> int:
    """Device bytes of cache_evict's workspace; needs no GPU."""
    return lib().mtb_cache_evict_workspace(int(n_seq), int(n_kv_heads), int(table_stride))


def cache_evict(cache: PagedCache, keep: int, new_len, workspace, sinks: int = 0, recent: int = 0, stream=None):
    """Keep the `keep` slots of each longer sequence that rank highest, in place (mtb_cache_evict); new_len int32 [sequences]
    gets the lengths (it may be kv_len itself)."""
    dev = cache.device
    wp, wn = _space(workspace, dev)
    rc = lib().mtb_cache_evict(cache.view, keep, sinks, recent, _flat(new_len, "new_len", "int32", cache.n_seq, dev), wp, wn,
                               _stream(dev, stream))
    if rc != 0:
        _ok(rc, "cache_evict")


def logits_process(logits, out=None, choice=None, history=None, hist_begin=None, hist_end=None, repetition=None, presence=None,
                   frequency=None, bias_ids=None, bias_values=None, bias_begin=None, bias_end=None, mask=None, mask_row=None,
                   stream=None):
    """Penalties, biases and masks on logits [rows][vocab], and the greedy choice (mtb_logits_process).  Row r's history is
    history[hist_begin[r]:hist_end[r]], its biases likewise; mask int32 or uint32 [mask rows][words], bit i % 32 of word i / 32."""
    rows, vocab = _shape(logits, "logits", 2)
    name, dev, st = _NAME[logits.dtype], logits.get_device(), logits.stride()
    _need(name in _CODES and (st[1] == 1 or vocab == 1), "logits must be [rows][vocab] of float32, float16 or bfloat16, rows contiguous")
    op = os_ = 0
    if out is not None:
        _need(out.shape == logits.shape and out.dtype == logits.dtype and out.get_device() == dev,
              "out must have the shape, type and device of logits")
        os_, s1 = out.stride()
        _need(s1 == 1 or vocab == 1, "an out row must be contiguous")
        op, os_ = out.data_ptr(), (os_ if rows > 1 else max(os_, vocab))
    mp = ms = mn = 0
    if mask is not None:
        mn, words = _shape(mask, "mask", 2)
        ms, s1 = mask.stride()
        _need(_NAME[mask.dtype] in ("int32", "uint32") and s1 == 1 and mask.get_device() == dev and words * 32 >= vocab
              and (mask_row is not None or mn >= rows),
              "mask must be int32 [mask rows][vocab / 32 words], with a row for each logits row or mask_row given")
        mp, ms = mask.data_ptr(), (ms if mn > 1 else max(ms, words))
    n_hist = 0 if history is None else history.numel()
    n_bias = 0 if bias_ids is None else bias_ids.numel()
    p = _PACK_LOGITS(_flat(history, "history", "int32", 0, dev), n_hist, _flat(hist_begin, "hist_begin", "int32", rows, dev),
                     _flat(hist_end, "hist_end", "int32", rows, dev), _flat(repetition, "repetition", "float32", rows, dev),
                     _flat(presence, "presence", "float32", rows, dev), _flat(frequency, "frequency", "float32", rows, dev),
                     _flat(bias_ids, "bias_ids", "int32", 0, dev), _flat(bias_values, "bias_values", "float32", n_bias, dev), n_bias,
                     _flat(bias_begin, "bias_begin", "int32", rows, dev), _flat(bias_end, "bias_end", "int32", rows, dev), mp, ms, mn,
                     _flat(mask_row, "mask_row", "int32", rows, dev))
    rc = lib().mtb_logits_process(logits.data_ptr(), _CODES[name], rows, vocab, st[0] if rows > 1 else max(st[0], vocab), p, op, os_,
                                  _flat(choice, "choice", "int32", rows, dev), _stream(dev, stream))
    if rc != 0:
        _ok(rc, "logits_process")
