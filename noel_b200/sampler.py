"""Python front end of libnoel_sampler_cuda.so (ctypes over the C ABI).

Mirrors the reference sampler's interface (Sain-Kai/noel include/sampler.h):
``Sampler`` wraps ``noel_sampler_t`` with the same init / set_config / sample
/ random_f32 / free semantics, and ``sample_batch`` exposes the batched
device entry point for torch tensors already on the GPU.  There is no CPU
path: loading fails loudly if the library has not been built.
"""
from __future__ import annotations

import ctypes as C
import os

import numpy as np

from .build import LIB

F32, BF16 = 0, 1
HEAD_F32, HEAD_F16, HEAD_BF16 = 0, 1, 30
ERR_INVALID_ARG = -1

STAT_NUM_CANDS, STAT_N_TOPK, STAT_N_FINAL, STAT_FLAGS = range(4)
ROW_GREEDY, ROW_EXACT_PASS, ROW_FALLBACK = 1, 2, 4


class SamplerConfig(C.Structure):
    """noel_sampler_config_t (include/sampler.h; reference include/sampler.h:12-19)."""

    _fields_ = [
        ("temperature", C.c_float),
        ("top_p", C.c_float),
        ("top_k", C.c_int),
        ("repetition_penalty", C.c_float),
        ("repetition_window", C.c_int),
        ("seed", C.c_uint64),
    ]


class TokenProb(C.Structure):
    _fields_ = [("id", C.c_int32), ("val", C.c_float)]


class SamplerStruct(C.Structure):
    """noel_sampler_t (reference include/sampler.h:26-31)."""

    _fields_ = [
        ("config", SamplerConfig),
        ("rng_state", C.c_uint64 * 2),
        ("candidates", C.POINTER(TokenProb)),
        ("candidate_capacity", C.c_int),
    ]


class Extras(C.Structure):
    _fields_ = [
        ("d_probs", C.c_void_p),
        ("d_list_ids", C.c_void_p),
        ("d_list_probs", C.c_void_p),
        ("list_len", C.c_int),
        ("list_weights", C.c_int),
        ("d_stats", C.c_void_p),
        ("write_back", C.c_int),
    ]


class NoelSamplerError(RuntimeError):
    def __init__(self, status: int, message: str):
        super().__init__(f"noel sampler status {status}: {message}")
        self.status = status


_lib = None


def lib() -> C.CDLL:
    """Load the in-tree library (raises if it has not been built)."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB):
        raise FileNotFoundError(f"{LIB} is missing: run `python -m noel_b200.build`")
    L = C.CDLL(LIB)
    L.noel_sampler_init.restype = None
    L.noel_sampler_init.argtypes = [C.POINTER(SamplerStruct), C.POINTER(SamplerConfig), C.c_int]
    L.noel_sampler_free.restype = None
    L.noel_sampler_free.argtypes = [C.POINTER(SamplerStruct)]
    L.noel_sampler_set_config.restype = None
    L.noel_sampler_set_config.argtypes = [C.POINTER(SamplerStruct), C.POINTER(SamplerConfig)]
    L.noel_sampler_sample.restype = C.c_int32
    L.noel_sampler_sample.argtypes = [C.POINTER(SamplerStruct), C.c_void_p, C.c_int, C.c_void_p, C.c_int]
    L.noel_sampler_random_f32.restype = C.c_float
    L.noel_sampler_random_f32.argtypes = [C.POINTER(SamplerStruct)]
    L.noel_sampler_sample_batch.restype = C.c_int
    L.noel_sampler_sample_batch.argtypes = [
        C.POINTER(SamplerConfig), C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_size_t, C.c_void_p,
        C.c_int, C.c_size_t, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p,
    ]
    L.noel_sampler_sample_batch_ex.restype = C.c_int
    L.noel_sampler_sample_batch_ex.argtypes = [
        C.POINTER(SamplerConfig), C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_size_t, C.c_void_p,
        C.c_int, C.c_size_t, C.c_void_p, C.c_void_p, C.POINTER(Extras), C.c_void_p,
    ]
    L.noel_sampler_sample_batch_host.restype = C.c_int
    L.noel_sampler_sample_batch_host.argtypes = [
        C.POINTER(SamplerConfig), C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_size_t, C.c_void_p,
        C.c_int, C.c_size_t, C.c_void_p, C.c_void_p, C.c_void_p,
    ]
    L.noel_sampler_shard_list_len.restype = C.c_int
    L.noel_sampler_shard_list_len.argtypes = [C.POINTER(SamplerConfig)]
    L.noel_sampler_shard_select.restype = C.c_int
    L.noel_sampler_shard_select.argtypes = [
        C.POINTER(SamplerConfig), C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_size_t, C.c_int,
        C.c_void_p, C.c_int, C.c_size_t, C.c_void_p, C.c_void_p,
    ]
    L.noel_sampler_shard_merge.restype = C.c_int
    L.noel_sampler_shard_merge.argtypes = [
        C.POINTER(SamplerConfig), C.c_int, C.c_int, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p,
        C.c_void_p, C.c_void_p,
    ]
    L.noel_postreq_sample_batch.restype = C.c_int
    L.noel_postreq_sample_batch.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_size_t, C.c_void_p,
                                            C.c_void_p, C.c_void_p]
    L.noel_postreq_apply_penalties_batch.restype = C.c_int
    L.noel_postreq_apply_penalties_batch.argtypes = [C.c_void_p, C.c_int, C.c_int, C.c_size_t, C.c_void_p, C.c_int,
                                                     C.c_size_t, C.c_float, C.c_int, C.c_void_p]
    L.noel_postreq_grammar_mask_batch.restype = C.c_int
    L.noel_postreq_grammar_mask_batch.argtypes = [C.c_void_p, C.c_int, C.c_int, C.c_size_t, C.c_void_p, C.c_int,
                                                  C.c_void_p]
    L.noel_postreq_sample.restype = C.c_int32
    L.noel_postreq_sample.argtypes = [C.c_void_p, C.c_int, C.c_void_p]
    L.noel_lmhead_sample.restype = C.c_int
    L.noel_lmhead_sample.argtypes = [C.POINTER(SamplerConfig), C.c_void_p, C.c_int, C.c_size_t, C.c_void_p,
                                     C.c_size_t, C.c_int, C.c_int, C.c_int, C.c_void_p, C.c_int, C.c_size_t,
                                     C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p]
    L.noel_lmhead_sample_ex.restype = C.c_int
    L.noel_lmhead_sample_ex.argtypes = [C.POINTER(SamplerConfig), C.c_void_p, C.c_int, C.c_size_t, C.c_void_p,
                                        C.c_size_t, C.c_int, C.c_int, C.c_int, C.c_void_p, C.c_void_p, C.c_void_p,
                                        C.c_void_p, C.c_int, C.c_size_t, C.c_void_p, C.c_void_p, C.c_void_p,
                                        C.c_void_p, C.c_void_p, C.c_size_t, C.c_void_p]
    L.noel_logits_process.restype = C.c_int
    L.noel_logits_process.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_size_t, C.c_void_p]
    L.noel_lora_workspace_bytes.restype = C.c_size_t
    L.noel_lora_workspace_bytes.argtypes = [C.c_int, C.c_int]
    L.noel_lora_apply.restype = C.c_int
    L.noel_lora_apply.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t, C.c_int, C.c_int, C.c_int,
                                  C.c_void_p, C.c_size_t, C.c_void_p, C.c_size_t, C.c_void_p]
    L.noel_moe_route_top_k.restype = C.c_int
    L.noel_moe_route_top_k.argtypes = [C.c_void_p, C.c_int, C.c_int, C.c_size_t, C.c_int, C.c_void_p, C.c_void_p]
    L.noel_sampler_cuda_last_error.restype = C.c_int
    L.noel_sampler_cuda_last_error_message.restype = C.c_char_p
    L.noel_sampler_cuda_status_string.restype = C.c_char_p
    L.noel_sampler_cuda_status_string.argtypes = [C.c_int]
    L.noel_sampler_cuda_expf_table_size.restype = C.c_int
    L.noel_sampler_cuda_profile_events.restype = C.c_int
    L.noel_sampler_cuda_profile_events.argtypes = [C.c_void_p, C.c_void_p]
    L.noel_sampler_cuda_expf_checksums.restype = C.c_int
    L.noel_sampler_cuda_expf_checksums.argtypes = [C.c_int, C.c_void_p, C.c_void_p]
    L.noel_sampler_cuda_sync_check.restype = C.c_int
    L.noel_sampler_cuda_sync_check.argtypes = [C.c_void_p]
    L.noel_sampler_cuda_set_wait_limit.restype = C.c_int
    L.noel_sampler_cuda_set_wait_limit.argtypes = [C.c_longlong, C.c_int]
    _lib = L
    return L


def _check(status: int) -> None:
    if status != 0:
        msg = lib().noel_sampler_cuda_last_error_message().decode(errors="replace")
        raise NoelSamplerError(status, msg)


def make_config(temperature=0.7, top_p=0.9, top_k=40, repetition_penalty=1.1,
                repetition_window=64, seed=0) -> SamplerConfig:
    return SamplerConfig(float(temperature), float(top_p), int(top_k), float(repetition_penalty),
                         int(repetition_window), int(seed))


class Sampler:
    """One noel_sampler_t, driven through the reference ABI."""

    def __init__(self, cfg: SamplerConfig | None = None, max_vocab: int = 1024):
        self.s = SamplerStruct()
        lib().noel_sampler_init(C.byref(self.s), C.byref(cfg) if cfg is not None else None, max_vocab)

    @property
    def config(self) -> SamplerConfig:
        return self.s.config

    @property
    def rng_state(self) -> tuple[int, int]:
        return (self.s.rng_state[0], self.s.rng_state[1])

    @rng_state.setter
    def rng_state(self, st) -> None:
        self.s.rng_state[0], self.s.rng_state[1] = int(st[0]), int(st[1])

    def set_config(self, cfg: SamplerConfig) -> None:
        lib().noel_sampler_set_config(C.byref(self.s), C.byref(cfg))

    def random_f32(self) -> float:
        return lib().noel_sampler_random_f32(C.byref(self.s))

    def sample(self, logits, history=None) -> int:
        """logits: float32 numpy array (host, modified in place when the
        penalty applies) or a CUDA torch tensor; history: int32 array/tensor."""
        lp, V = _ptr_len(logits)
        hp, H = _ptr_len(history) if history is not None else (None, 0)
        r = lib().noel_sampler_sample(C.byref(self.s), lp, V, hp, H)
        st = lib().noel_sampler_cuda_last_error()
        if st != 0:
            _check(st)
        return int(r)

    def candidates(self, n: int) -> list[tuple[int, float]]:
        return [(self.s.candidates[i].id, self.s.candidates[i].val) for i in range(n)]

    def free(self) -> None:
        lib().noel_sampler_free(C.byref(self.s))

    def __del__(self):
        try:
            if self.s.candidates:
                self.free()
        except Exception:
            pass


def _ptr_len(a):
    if a is None:
        return None, 0
    if isinstance(a, np.ndarray):
        assert a.flags.c_contiguous
        return a.ctypes.data, a.size
    return a.data_ptr(), a.numel()  # torch tensor


def sample_batch(logits, rng, cfg: SamplerConfig, history=None, probs: bool = True,
                 list_len: int = 0, list_weights: bool = False, stats: bool = False,
                 write_back: bool = False, vocab: int | None = None, stream=None):
    """Batched device sampling of torch tensors on the current CUDA device.

    logits: [B, ld] float32 or bfloat16 (row stride ld >= vocab, unit column
    stride); rng: [B, 2] int64 xorshift128+ states, advanced in place;
    history: [B, hld] int32 or None.  Returns a dict of torch tensors:
    ids [B] int32, and as requested probs [B], list_ids/list_probs
    [B, list_len], stats [B, 4].
    """
    import torch

    assert logits.is_cuda and logits.dim() == 2 and logits.stride(1) == 1
    B, ld = logits.shape[0], logits.stride(0)
    V = logits.shape[1] if vocab is None else vocab
    dtype = {torch.float32: F32, torch.bfloat16: BF16}[logits.dtype]
    assert rng.dtype == torch.int64 and rng.shape == (B, 2) and rng.is_contiguous()
    dev = logits.device
    out = {"ids": torch.empty(B, dtype=torch.int32, device=dev)}
    ex = Extras()
    if probs:
        out["probs"] = torch.empty(B, dtype=torch.float32, device=dev)
        ex.d_probs = out["probs"].data_ptr()
    if list_len:
        out["list_ids"] = torch.empty(B, list_len, dtype=torch.int32, device=dev)
        out["list_probs"] = torch.empty(B, list_len, dtype=torch.float32, device=dev)
        ex.d_list_ids = out["list_ids"].data_ptr()
        ex.d_list_probs = out["list_probs"].data_ptr()
        ex.list_len = list_len
        ex.list_weights = 1 if list_weights else 0
    if stats:
        out["stats"] = torch.empty(B, 4, dtype=torch.int32, device=dev)
        ex.d_stats = out["stats"].data_ptr()
    ex.write_back = 1 if write_back else 0
    if history is not None:
        assert history.is_cuda and history.dtype == torch.int32 and history.stride(1) == 1
        hp, H, hld = history.data_ptr(), history.shape[1], history.stride(0)
    else:
        hp, H, hld = None, 0, 0
    s = stream if stream is not None else torch.cuda.current_stream(dev)
    _check(lib().noel_sampler_sample_batch_ex(C.byref(cfg), logits.data_ptr(), dtype, B, V, ld, hp, H, hld,
                                              rng.data_ptr(), out["ids"].data_ptr(), C.byref(ex),
                                              C.c_void_p(s.cuda_stream)))
    return out


def sample_batch_raw(cfg: SamplerConfig, logits_ptr: int, dtype: int, B: int, V: int, ld: int,
                     hist_ptr, H: int, hld: int, rng_ptr: int, ids_ptr: int, probs_ptr, stream_ptr) -> None:
    """Thin pass-through to noel_sampler_sample_batch (pointers as ints)."""
    _check(lib().noel_sampler_sample_batch(C.byref(cfg), logits_ptr, dtype, B, V, ld, hist_ptr, H, hld,
                                           rng_ptr, ids_ptr, probs_ptr, C.c_void_p(stream_ptr)))


def sample_batch_host(cfg: SamplerConfig, logits: np.ndarray, rng: np.ndarray, history: np.ndarray | None = None,
                      probs: bool = False, vocab: int | None = None):
    """Host-buffer batched sampling (noel_sampler_sample_batch_host).
    logits: [B, ld] float32, or uint16 holding bf16 bits; rng [B, 2] uint64
    (advanced in place).  Returns ids (and probs)."""
    B, ld = logits.shape
    V = ld if vocab is None else vocab
    dtype = BF16 if logits.dtype == np.uint16 else F32
    assert logits.flags.c_contiguous and rng.flags.c_contiguous and rng.dtype == np.uint64
    ids = np.empty(B, np.int32)
    pr = np.empty(B, np.float32) if probs else None
    if history is not None:
        assert history.dtype == np.int32 and history.flags.c_contiguous
        hp, H, hld = history.ctypes.data, history.shape[1], history.shape[1]
    else:
        hp, H, hld = None, 0, 0
    _check(lib().noel_sampler_sample_batch_host(C.byref(cfg), logits.ctypes.data, dtype, B, V, ld, hp, H, hld,
                                                rng.ctypes.data, ids.ctypes.data,
                                                pr.ctypes.data if pr is not None else None))
    return (ids, pr) if probs else ids


def profile_events(before=None, after=None) -> None:
    """Record torch.cuda.Event ``before``/``after`` around the single-pass
    kernel of later batched calls on this thread (None, None to stop)."""
    for ev in (before, after):
        if ev is not None and not ev.cuda_event:
            ev.record()  # torch creates the CUDA event on its first record
    lib().noel_sampler_cuda_profile_events(before.cuda_event if before is not None else None,
                                           after.cuda_event if after is not None else None)


def sync_check(stream=None) -> int:
    """Wait for ``stream`` (default: the current one) and return the status of
    the device-side waits of the calls made on it (0, or NOEL_ERR_DEVICE_WAIT)."""
    import torch

    s = stream if stream is not None else torch.cuda.current_stream()
    return int(lib().noel_sampler_cuda_sync_check(C.c_void_p(s.cuda_stream)))


def set_wait_limit(wait_ns: int = 0, stall_next_call: bool = False) -> None:
    """Limit of the device-side waits of this thread's later batched calls
    (0: the default, 2 s); ``stall_next_call`` makes the next call's kernel
    issue no row loads so that its waits run out (failure-detection tests)."""
    _check(lib().noel_sampler_cuda_set_wait_limit(int(wait_ns), 1 if stall_next_call else 0))


def expf_table_size() -> int:
    return lib().noel_sampler_cuda_expf_table_size()


def expf_checksums(chunk_log2: int = 24):
    """Device exp-weight checksums over (-15, 0] (see include/noel_sampler_cuda.h)."""
    import torch

    n = -(-(0xC1700000 - 0x80000000) // (1 << chunk_log2))
    out = torch.empty(n, dtype=torch.int64, device="cuda")
    s = torch.cuda.current_stream()
    _check(lib().noel_sampler_cuda_expf_checksums(chunk_log2, out.data_ptr(), C.c_void_p(s.cuda_stream)))
    s.synchronize()
    return out.cpu().numpy().view(np.uint64)


def route_top_k(gate_logits, top_k: int):
    """MoE routing of every row of gate_logits (a CUDA float32 tensor [T, E],
    unit column stride): the reference's aether_route_top_k per token.
    Returns (expert ids [T, top_k] int32, weights [T, top_k] float32)."""
    import torch

    assert gate_logits.is_cuda and gate_logits.dtype == torch.float32 and gate_logits.stride(1) == 1
    T, E = gate_logits.shape
    out = torch.empty(T, top_k, 2, dtype=torch.int32, device=gate_logits.device)
    s = torch.cuda.current_stream(gate_logits.device)
    _check(lib().noel_moe_route_top_k(gate_logits.data_ptr(), T, E, gate_logits.stride(0), top_k, out.data_ptr(),
                                      C.c_void_p(s.cuda_stream)))
    return out[:, :, 0], out[:, :, 1].view(torch.float32)


class PostreqParams(C.Structure):
    """noel_postreq_params_t (include/noel_postreq.h; the reference's
    aether_sampling_params_t, include/pipeline_stages.h:13-20)."""

    _fields_ = [("temperature", C.c_float), ("top_p", C.c_float), ("top_k", C.c_int),
                ("repetition_penalty", C.c_float), ("repetition_window", C.c_int),
                ("grammar_enforce_json", C.c_bool)]


def postreq_params(temperature=0.7, top_p=0.9, top_k=50, repetition_penalty=1.15, repetition_window=2048,
                   grammar_enforce_json=False) -> PostreqParams:
    return PostreqParams(temperature, top_p, top_k, repetition_penalty, repetition_window, grammar_enforce_json)


def postreq_sample_batch(logits, params: PostreqParams, uniforms):
    """aether_postreq_sample on every row of logits (CUDA float32 [B, V],
    unit column stride; modified in place as the reference modifies its row)
    with the rows' uniforms (CUDA float32 [B]).  Returns ids [B] int32."""
    import torch

    assert logits.is_cuda and logits.dtype == torch.float32 and logits.stride(1) == 1
    B, V = logits.shape
    ids = torch.empty(B, dtype=torch.int32, device=logits.device)
    s = torch.cuda.current_stream(logits.device)
    _check(lib().noel_postreq_sample_batch(C.byref(params), logits.data_ptr(), B, V, logits.stride(0),
                                           uniforms.data_ptr() if uniforms is not None else None, ids.data_ptr(),
                                           C.c_void_p(s.cuda_stream)))
    return ids


def postreq_apply_penalties_batch(logits, history, penalty: float, window: int) -> None:
    import torch

    B, V = logits.shape
    s = torch.cuda.current_stream(logits.device)
    _check(lib().noel_postreq_apply_penalties_batch(logits.data_ptr(), B, V, logits.stride(0), history.data_ptr(),
                                                    history.shape[1], history.stride(0), penalty, window,
                                                    C.c_void_p(s.cuda_stream)))


def postreq_grammar_mask_batch(logits, states=None, state: int = 0) -> None:
    import torch

    B, V = logits.shape
    s = torch.cuda.current_stream(logits.device)
    _check(lib().noel_postreq_grammar_mask_batch(logits.data_ptr(), B, V, logits.stride(0),
                                                 states.data_ptr() if states is not None else None, state,
                                                 C.c_void_p(s.cuda_stream)))


def postreq_sample(logits, params: PostreqParams) -> int:
    """The drop-in single-row call (host numpy float32 row or CUDA tensor),
    drawing rand() where the reference does."""
    lp, V = _ptr_len(logits)
    r = lib().noel_postreq_sample(lp, V, C.byref(params))
    st = lib().noel_sampler_cuda_last_error()
    if st != 0:
        _check(st)
    return int(r)


def _refuse(message: str):
    raise NoelSamplerError(ERR_INVALID_ARG, message)


def _on(tensor, dtype, shape, name: str, device):
    """tensor's address after the checks every argument gets: on device, of
    dtype, of shape (None: any extent), its last axis of unit stride."""
    if tensor is None:
        return None
    if tensor.dtype is not dtype:
        _refuse(f"{name}: {dtype} wanted, got {tensor.dtype}")
    if not tensor.is_cuda:
        _refuse(f"{name} is not on a GPU")
    if tensor.get_device() != device.index:
        _refuse(f"{name} is on {tensor.device}, {device} wanted")
    have = tensor.shape
    if len(have) != len(shape):
        _refuse(f"{name}: shape {tuple(shape)} wanted, got {tuple(have)}")
    for w, h in zip(shape, have):
        if w is not None and w != h:
            _refuse(f"{name}: shape {tuple(shape)} wanted, got {tuple(have)}")
    if have[-1] > 1 and tensor.stride(-1) != 1:
        _refuse(f"{name}: its last axis must be contiguous")
    return tensor.data_ptr()


def _pitch(tensor, axis: int = 0) -> int:
    """Elements from one index of axis to the next; where there is only one
    (its stride may be anything), the last axis's extent."""
    return tensor.stride(axis) if tensor.shape[axis] > 1 else tensor.shape[-1]


def _own_pitch(tensor, axis: int = 0) -> int:
    """_pitch, but a single one keeps its stride where rows may have it: the
    adapters' kernels go by the alignment of pitches, and a view of one row is
    taken as the row is among others."""
    return max(tensor.stride(axis), tensor.shape[-1]) if tensor.shape[axis] == 1 else tensor.stride(axis)


def _row_values(tensor, dtype, batch, name: str, device):
    """The address of one value a row (or adapter)."""
    return _on(tensor, dtype, (batch,), name, device)


def _call(device, stream, run) -> None:
    """run(stream address) with device the current one, on stream or on the
    device's current stream; raises on a status that is not 0."""
    import torch

    index = device.index
    before = torch._C._cuda_getDevice()
    if before != index:
        torch.cuda.set_device(index)
    try:
        status = run(stream.cuda_stream if stream is not None else torch._C._cuda_getCurrentRawStream(index))
    finally:
        if before != index:
            torch.cuda.set_device(before)
    if status != 0:
        _check(status)


class LogitsParamsStruct(C.Structure):
    """noel_logits_params_t (include/noel_logits.h)."""

    _fields_ = [("d_history", C.c_void_p), ("hld", C.c_size_t), ("history_len", C.c_int),
                ("d_history_lens", C.c_void_p), ("d_prompt_lens", C.c_void_p), ("d_repetition", C.c_void_p),
                ("d_frequency", C.c_void_p), ("d_presence", C.c_void_p), ("d_bias_ids", C.c_void_p),
                ("d_bias", C.c_void_p), ("bld", C.c_size_t), ("bias_len", C.c_int), ("d_mask", C.c_void_p),
                ("mld", C.c_size_t), ("mask_rows", C.c_int), ("d_mask_rows", C.c_void_p), ("v_begin", C.c_int)]


class LogitsParams:
    """What ``logits_process`` applies to each row of a batch of B rows
    (include/noel_logits.h); every part may be left out.

    history [B, H] int32 token ids, its first history_lens [B] int32 used and
    the first prompt_lens [B] int32 of them the prompt; repetition, frequency,
    presence [B] float32; bias_ids [B, N] int32 with bias [B, N] float32; mask
    [M, words] int32, bit v % 32 of word v // 32 set where id v is allowed, and
    mask_rows [B] int32 the mask of each row (outside 0 .. M - 1: none; left
    out: mask b for row b); v_begin the id of the logits' first column.

    The object holds the tensors themselves: a serving loop makes it once over
    its buffers and writes the next step's values into them.
    """

    def __init__(self, history=None, history_lens=None, prompt_lens=None, repetition=None, frequency=None,
                 presence=None, bias_ids=None, bias=None, mask=None, mask_rows=None, v_begin: int = 0):
        import torch

        self.tensors = [t for t in (history, history_lens, prompt_lens, repetition, frequency, presence, bias_ids,
                                    bias, mask, mask_rows) if t is not None]
        self.device = self.tensors[0].device if self.tensors else None
        dev = self.device
        if (bias_ids is None) != (bias is None):
            _refuse("bias_ids and bias come together")
        if history is None and any(t is not None for t in (history_lens, prompt_lens)):
            _refuse("history_lens and prompt_lens need a history")
        if mask is None and mask_rows is not None:
            _refuse("mask_rows needs a mask")
        per_row = [t for t in (history, history_lens, prompt_lens, repetition, frequency, presence, bias_ids, bias,
                               mask_rows) if t is not None]
        self.batch = per_row[0].shape[0] if per_row and per_row[0].dim() else None
        B, i32, f32 = self.batch, torch.int32, torch.float32
        s = self.s = LogitsParamsStruct()
        s.d_history = _on(history, i32, (B, None), "history", dev)
        s.d_history_lens = _row_values(history_lens, i32, B, "history_lens", dev)
        s.d_prompt_lens = _row_values(prompt_lens, i32, B, "prompt_lens", dev)
        s.d_repetition = _row_values(repetition, f32, B, "repetition", dev)
        s.d_frequency = _row_values(frequency, f32, B, "frequency", dev)
        s.d_presence = _row_values(presence, f32, B, "presence", dev)
        if history is not None:
            s.hld, s.history_len = _pitch(history), history.shape[1]
        if bias_ids is not None:
            s.d_bias_ids = _on(bias_ids, i32, (B, None), "bias_ids", dev)
            s.d_bias = _on(bias, f32, tuple(bias_ids.shape), "bias", dev)
            s.bld, s.bias_len = _pitch(bias_ids), bias_ids.shape[1]
            if _pitch(bias) != s.bld:
                _refuse("bias and bias_ids need rows of the same pitch")
        if mask is not None:
            s.d_mask = _on(mask, i32, (None, None), "mask", dev)
            s.mld, s.mask_rows = _pitch(mask), mask.shape[0]
            s.d_mask_rows = _row_values(mask_rows, i32, B, "mask_rows", dev)
            self.words = mask.shape[1]
        if not 0 <= v_begin < 2**31:  # ctypes would keep its lowest 32 bits
            _refuse(f"v_begin {v_begin}")
        s.v_begin = v_begin
        self.ref = C.byref(s)

    def check(self, logits, vocab: int) -> None:
        """Whether these parameters fit rows of logits of vocab columns."""
        if self.tensors and self.device != logits.device:
            _refuse(f"parameters on {self.device}, logits on {logits.device}")
        if self.batch is not None and self.batch != logits.shape[0]:
            _refuse(f"parameters for {self.batch} rows, logits of {logits.shape[0]}")
        if self.s.d_mask and self.words * 32 < self.s.v_begin + vocab:
            _refuse(f"masks of {self.words} words for ids up to {self.s.v_begin + vocab - 1}")


def logits_process(logits, params: LogitsParams, vocab: int | None = None, stream=None):
    """Penalties, biases and masks on every row of logits, in place
    (include/noel_logits.h): logits [B, ld] CUDA float32 or bfloat16 with unit
    column stride, of which the first vocab columns (default: all) hold the
    ids from params.v_begin on.  Returns logits."""
    import torch

    dtype = {torch.float32: F32, torch.bfloat16: BF16}.get(logits.dtype)
    if dtype is None:
        _refuse(f"logits: float32 or bfloat16 wanted, got {logits.dtype}")
    dev = logits.device
    ptr = _on(logits, logits.dtype, (None, None), "logits", dev)
    B, cols = logits.shape
    V = cols if vocab is None else vocab
    if not 0 < V <= cols:
        _refuse(f"vocab {V} of {cols} columns")
    params.check(logits, V)
    _call(dev, stream, lambda s: lib().noel_logits_process(params.ref, ptr, dtype, B, V, _pitch(logits), s))
    return logits


class LoraStruct(C.Structure):
    """noel_lora_t (include/noel_lora.h)."""

    _fields_ = [("d_a", C.c_void_p), ("lda", C.c_size_t), ("stride_a", C.c_size_t), ("d_b", C.c_void_p),
                ("ldb", C.c_size_t), ("stride_b", C.c_size_t), ("d_scale", C.c_void_p), ("d_ranks", C.c_void_p),
                ("type", C.c_int), ("n_adapters", C.c_int), ("rank", C.c_int)]


class Adapters:
    """n low-rank adapters of one weight [V, D] (include/noel_lora.h): adapter
    i is scale[i] * b[i] @ a[i] with a [n, r, D] and b [n, V, r], both float32,
    float16 or bfloat16; scale [n] float32 (default 1) and ranks [n] int32
    (adapters of a smaller rank than r).  Holds the tensors themselves."""

    def __init__(self, a, b, scale=None, ranks=None):
        import torch

        kind = {torch.float32: HEAD_F32, torch.float16: HEAD_F16, torch.bfloat16: HEAD_BF16}.get(a.dtype)
        if kind is None:
            _refuse(f"a: float32, float16 or bfloat16 wanted, got {a.dtype}")
        self.device, self.tensors = a.device, (a, b, scale, ranks)
        s = self.s = LoraStruct()
        s.d_a = _on(a, a.dtype, (None, None, None), "a", a.device)
        self.n, self.rank, self.cols = a.shape
        s.d_b = _on(b, a.dtype, (self.n, None, self.rank), "b", a.device)
        self.rows = b.shape[1]
        s.lda, s.stride_a, s.ldb, s.stride_b = _own_pitch(a, 1), _own_pitch(a), _own_pitch(b, 1), _own_pitch(b)
        s.d_scale = _row_values(scale, torch.float32, self.n, "scale", a.device)
        s.d_ranks = _row_values(ranks, torch.int32, self.n, "ranks", a.device)
        s.type, s.n_adapters, s.rank = kind, self.n, self.rank
        self.ref, self.sizes = C.byref(s), {}

    def scratch(self, batch: int):
        """Scratch of one call over batch tokens (None where it needs none) and its bytes."""
        import torch

        size = self.sizes.get(batch)
        if size is None:
            size = self.sizes[batch] = lib().noel_lora_workspace_bytes(batch, self.rank)
        return (torch.empty(size, dtype=torch.uint8, device=self.device) if size else None), size


def lora_apply(y, x, adapters: Adapters, adapter_ids, stream=None):
    """y[t] += scale[i] * b[i] @ (a[i] @ x[t]) in place, i = adapter_ids[t]
    (outside 0 .. n - 1: y[t] is left as it is): y [B, V] and x [B, D] CUDA
    float32 with unit column stride, adapter_ids [B] int32.  Returns y."""
    import torch

    dev = adapters.device
    yp = _on(y, torch.float32, (None, adapters.rows), "y", dev)
    B = y.shape[0]
    xp = _on(x, torch.float32, (B, adapters.cols), "x", dev)
    ip = _row_values(adapter_ids, torch.int32, B, "adapter_ids", dev)
    if stream is None:
        work, size = adapters.scratch(B)
    else:
        with torch.cuda.stream(stream):
            work, size = adapters.scratch(B)
    _call(dev, stream, lambda s: lib().noel_lora_apply(adapters.ref, ip, xp, _own_pitch(x), B, adapters.cols, adapters.rows,
                                                       yp, _own_pitch(y), work.data_ptr() if size else None, size, s))
    return y


def lmhead_sample(weight, hidden, rng, cfg: SamplerConfig, history=None, probs: bool = False,
                  adapters: Adapters | None = None, adapter_ids=None, process: LogitsParams | None = None):
    """The LM head then the sampler (include/noel_lmhead.h): weight [V, D]
    CUDA float32 / float16 / bfloat16 (unit column stride), hidden [B, D]
    CUDA float32, rng [B, 2] int64 advanced in place, history [B, H] int32 or
    None.  adapters with adapter_ids [B] int32 add each token's low-rank part
    to its logits, and process is applied to them before sampling.  Returns
    (ids [B] int32, logits [B, V] float32, probs or None)."""
    import torch

    wt = {torch.float32: HEAD_F32, torch.float16: HEAD_F16, torch.bfloat16: HEAD_BF16}[weight.dtype]
    dev = weight.device
    wp = _on(weight, weight.dtype, (None, None), "weight", dev)
    V, D = weight.shape
    xp = _on(hidden, torch.float32, (None, D), "hidden", dev)
    B = hidden.shape[0]
    gp = _on(rng, torch.int64, (B, 2), "rng", dev)
    if not rng.is_contiguous():
        _refuse("rng: rows side by side wanted")
    if (adapters is None) != (adapter_ids is None):
        _refuse("adapters and adapter_ids come together")
    logits = torch.empty(B, V, dtype=torch.float32, device=dev)
    ids = torch.empty(B, dtype=torch.int32, device=dev)
    pr = torch.empty(B, dtype=torch.float32, device=dev) if probs else None
    if history is not None:
        hp, H, hld = _on(history, torch.int32, (B, None), "history", dev), history.shape[1], _pitch(history)
    else:
        hp, H, hld = None, 0, 0
    lora = ip = work = None
    size = 0
    if adapters is not None:
        if adapters.device != dev or (adapters.rows, adapters.cols) != (V, D):
            _refuse(f"adapters of a [{adapters.rows}, {adapters.cols}] weight on {adapters.device}, "
                    f"the head is [{V}, {D}] on {dev}")
        lora, ip = adapters.ref, _row_values(adapter_ids, torch.int32, B, "adapter_ids", dev)
        work, size = adapters.scratch(B)
    if process is not None:
        process.check(logits, V)
    _call(dev, None, lambda s: lib().noel_lmhead_sample_ex(
        C.byref(cfg), wp, wt, _pitch(weight), xp, _own_pitch(hidden), B, D, V, lora, ip,
        process.ref if process is not None else None, hp, H, hld, gp, ids.data_ptr(),
        pr.data_ptr() if pr is not None else None, logits.data_ptr(), work.data_ptr() if size else None, size, s))
    return ids, logits, pr
