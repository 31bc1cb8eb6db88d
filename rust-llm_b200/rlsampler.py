"""ctypes front end of librl_sampler.so (include/rl_sampler.h).

Device buffers are torch tensors (torch is used only for device memory and
streams); every call goes through the C ABI. There is no fallback: if the
shared library is missing or fails to load, import of the sampler fails.
"""
from __future__ import annotations

import ctypes
import os
import re

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
LIB_PATH = os.path.join(HERE, "librl_sampler.so")
HEADER = os.path.join(ROOT, "include", "rl_sampler.h")

RL_OK = 0
RL_ERR_INVALID_ARG = 1
RL_ERR_SHAPE = 2
RL_ERR_OOM = 3
RL_ERR_CUDA = 4
RL_ERR_NCCL = 5
RL_ERR_TIMEOUT = 6
RL_ERR_UNSUPPORTED = 7
RL_ERR_NONFINITE = 8
RL_F32 = 0
RL_BF16 = 1
RL_DEBUG_EXPIRE_WAIT = 1
RL_DEBUG_TIMING = 2
RL_CREATE_SHARDED = 1
NCCL_ID_BYTES = 128  # RL_NCCL_ID_BYTES

PART_KEYS = 128  # RL_PART_KEYS
PART_REC = PART_KEYS + 4  # u64 words of a packed partial record (keys, then rl_part_stats)
PART_STATS_DTYPE = np.dtype(
    [
        ("m", np.float32),
        ("argmax", np.int32),
        ("nallow", np.int32),
        ("flags", np.int32),
        ("z", np.float64),
        ("n", np.int32),
        ("pad", np.int32),
    ]
)

STATUS_NAMES = {0: "OK", 1: "INVALID_ARG", 2: "SHAPE", 3: "OOM", 4: "CUDA", 5: "NCCL",
                6: "TIMEOUT", 7: "UNSUPPORTED", 8: "NONFINITE"}

ROW_PARAMS_DTYPE = np.dtype(
    [
        ("temperature", np.float32),
        ("top_p", np.float32),
        ("top_k", np.int32),
        ("repeat_penalty", np.float32),
        ("presence_penalty", np.float32),
        ("frequency_penalty", np.float32),
    ]
)


class _DistRows(ctypes.Structure):
    """rl_dist_rows."""

    _fields_ = [("logits", ctypes.c_void_p), ("dtype", ctypes.c_int), ("rows", ctypes.c_int32), ("ld", ctypes.c_int64),
                ("temperature", ctypes.c_void_p), ("mask", ctypes.c_void_p), ("mask_stride", ctypes.c_int64),
                ("cut", ctypes.c_void_p), ("cut_stride", ctypes.c_int64), ("first_row", ctypes.c_void_p)]


class _Q4Weight(ctypes.Structure):
    """rl_q4_weight."""

    _fields_ = [("q", ctypes.c_void_p), ("ldq", ctypes.c_int64), ("scale", ctypes.c_void_p), ("lds", ctypes.c_int64),
                ("group", ctypes.c_int32)]


VERIFY_MAX_NODES = 256  # RL_VERIFY_MAX_NODES


class RLError(RuntimeError):
    def __init__(self, status, msg):
        super().__init__(f"{STATUS_NAMES.get(status, status)}: {msg}")
        self.status = status


_lib = None


def declared_symbols():
    """Entry points declared in include/rl_sampler.h."""
    txt = open(HEADER).read()
    return sorted(set(re.findall(r"^\s*(?:rl_status|const char\*)\s+(rl_\w+)\s*\(", txt, re.M)))


def lib():
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RLError(RL_ERR_UNSUPPORTED, f"{LIB_PATH} is missing: run rust-llm_b200/build.py")
        L = ctypes.CDLL(LIB_PATH)
        P = ctypes.c_void_p
        I = ctypes.c_int
        I64 = ctypes.c_int64
        F = ctypes.c_float
        L.rl_last_error.restype = ctypes.c_char_p
        L.rl_last_error.argtypes = []
        L.rl_version.restype = ctypes.c_char_p
        L.rl_version.argtypes = []
        L.rl_sampler_create.restype = I
        L.rl_sampler_create.argtypes = [ctypes.POINTER(P), I, I, I, I, ctypes.c_uint32]
        L.rl_sampler_destroy.restype = I
        L.rl_sampler_destroy.argtypes = [P]
        L.rl_sample_batch.restype = I
        L.rl_sample_batch.argtypes = [P, P, I, I, I, I64, P, P, I, P, I64, P, P, P, P, P, P]
        L.rl_sample_batch_debug.restype = I
        L.rl_sample_batch_debug.argtypes = [P, P, I, I, I, I64, P, P, I, P, I64, P, P, P, P, P, P,
                                            P, P, I, P, P]
        L.rl_sample_batch_static.restype = I
        L.rl_sample_batch_static.argtypes = [P, I, I, I, I64, P, P, I, P, I64, P, P, P, P, P, P]
        L.rl_sample_host.restype = I
        L.rl_sample_host.argtypes = [P, P, I, I, P, P, I, P, I64, P, P, P, P]
        L.rl_decoder_sample.restype = I
        L.rl_decoder_sample.argtypes = [P, P, I, I, I64, P, P, P, P, P, P]
        L.rl_decoder_sample_host.restype = I
        L.rl_decoder_sample_host.argtypes = [P, P, I, I, P, P, P, P, P]
        L.rl_greedy.restype = I
        L.rl_greedy.argtypes = [P, P, I, I, I64, P, P]
        L.rl_grammar_greedy.restype = I
        L.rl_grammar_greedy.argtypes = [P, P, I, I, I64, P, I64, P, P]
        L.rl_specdec_sample.restype = I
        L.rl_specdec_sample.argtypes = [P, P, I, I, I64, P, P, P, P, P]
        L.rl_specdec_verify.restype = I
        L.rl_specdec_verify.argtypes = [P, P, I, I, I64, P, I, P, P, P, P, P, P, P]
        D = ctypes.POINTER(_DistRows)
        L.rl_specdec_verify_draft.restype = I
        L.rl_specdec_verify_draft.argtypes = [P, I, I, I, D, D, P, P, P, P, P, P, P, P, P]
        L.rl_specdec_verify_tree.restype = I
        L.rl_specdec_verify_tree.argtypes = [P, I, I, I, D, D, P, P, P, P, P, P, P, P, P, P, P]
        L.rl_greedy_host.restype = I
        L.rl_greedy_host.argtypes = [P, P, I, I, P]
        L.rl_grammar_greedy_host.restype = I
        L.rl_grammar_greedy_host.argtypes = [P, P, I, I, P, I64, P]
        L.rl_beam_step.restype = I
        L.rl_beam_step.argtypes = [P, P, I, I, I, I64, P, P, P, F, I, I, I, P, P, P, P, P]
        L.rl_sample_partial.restype = I
        L.rl_sample_partial.argtypes = [P, P, I, I, I, I64, I, P, P, I, P, I64, P, P, P, P]
        L.rl_sample_merge.restype = I
        L.rl_sample_merge.argtypes = [P, I, I, P, P, P, P, P, P, P, P]
        L.rl_sample_sharded.restype = I
        L.rl_sample_sharded.argtypes = [P, P, P, I, I, I, I64, I, I, P, P, I, P, I64, P, P, P, P, P, P]
        L.rl_nccl_unique_id.restype = I
        L.rl_nccl_unique_id.argtypes = [P]
        L.rl_nccl_comm_init.restype = I
        L.rl_nccl_comm_init.argtypes = [ctypes.POINTER(P), I, P, I]
        L.rl_nccl_comm_destroy.restype = I
        L.rl_nccl_comm_destroy.argtypes = [P]
        L.rl_sampler_kernel_times.restype = I
        L.rl_sampler_kernel_times.argtypes = [P, P, I, P]
        L.rl_sampler_set_debug.restype = I
        L.rl_sampler_set_debug.argtypes = [P, ctypes.c_uint32]
        L.rl_selfcheck_div.restype = I
        L.rl_selfcheck_div.argtypes = [P, I, P, I, P, P, P]
        L.rl_gbnf_create.restype = I
        L.rl_gbnf_create.argtypes = [ctypes.c_char_p, ctypes.c_char_p, I, P, P, ctypes.c_int32, ctypes.POINTER(P)]
        L.rl_gbnf_destroy.restype = None
        L.rl_gbnf_destroy.argtypes = [P]
        L.rl_gbnf_state_create.restype = I
        L.rl_gbnf_state_create.argtypes = [P, ctypes.POINTER(P)]
        L.rl_gbnf_state_destroy.restype = None
        L.rl_gbnf_state_destroy.argtypes = [P]
        L.rl_gbnf_state_copy.restype = I
        L.rl_gbnf_state_copy.argtypes = [P, P]
        L.rl_gbnf_accepting.restype = I
        L.rl_gbnf_accepting.argtypes = [P]
        L.rl_gbnf_accept.restype = I
        L.rl_gbnf_accept.argtypes = [P, P, ctypes.c_int32]
        L.rl_gbnf_mask.restype = I
        L.rl_gbnf_mask.argtypes = [P, P, P, I64, P]
        L.rl_gbnf_accept_batch.restype = I
        L.rl_gbnf_accept_batch.argtypes = [P, P, P, I, P, I]
        L.rl_gbnf_mask_batch.restype = I
        L.rl_gbnf_mask_batch.argtypes = [P, P, I, P, I64, P, I]
        L.rl_lmhead_logits.restype = I
        L.rl_lmhead_logits.argtypes = [P, P, I64, P, I64, I, I, I, P, I, I64, P]
        L.rl_lmhead_greedy.restype = I
        L.rl_lmhead_greedy.argtypes = [P, P, I64, P, I64, I, I, I, P, P, P, I64, P]
        L.rl_lmhead_sample.restype = I
        L.rl_lmhead_sample.argtypes = [P, P, I64, P, I64, I, I, I, P, P, I, P, P, P, P, P, P]
        W = ctypes.POINTER(_Q4Weight)
        L.rl_lmhead_q4_quantize.restype = I
        L.rl_lmhead_q4_quantize.argtypes = [P, P, I64, I, I, I, P, I64, P, I64, P]
        L.rl_lmhead_q4_logits.restype = I
        L.rl_lmhead_q4_logits.argtypes = [P, P, I64, W, I, I, I, P, I, I64, P]
        L.rl_lmhead_q4_greedy.restype = I
        L.rl_lmhead_q4_greedy.argtypes = [P, P, I64, W, I, I, I, P, P, P, I64, P]
        L.rl_lmhead_q4_sample.restype = I
        L.rl_lmhead_q4_sample.argtypes = [P, P, I64, W, I, I, I, P, P, I, P, P, P, P, P, P]
        _lib = L
    return _lib


def last_error() -> str:
    return lib().rl_last_error().decode()


def check(st, what=""):
    if st != RL_OK:
        raise RLError(st, f"{what}: {last_error()}")


def _ptr(t):
    """Device (or host numpy) pointer of a tensor/array, None for None."""
    if t is None:
        return None
    if isinstance(t, np.ndarray):
        return t.ctypes.data_as(ctypes.c_void_p)
    return ctypes.c_void_p(t.data_ptr())


def _stream(stream):
    if stream is None:
        import torch

        stream = torch.cuda.current_stream()
    return ctypes.c_void_p(stream.cuda_stream)


def _raw_stream(stream, device):
    """The stream's handle: the device's current stream where none is given
    (asked of torch without making a Stream object, where it can be)."""
    if stream is not None:
        return stream.cuda_stream
    import torch

    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    if raw is not None and device.index is not None:
        return raw(device.index)
    return torch.cuda.current_stream(device).cuda_stream


class DistRows:
    """Rows of distributions softmax(logits / T) over their kept ids
    (rl_dist_rows): logits [R, V] f32 or bf16, temperature [B] f32 (None: 1),
    mask [R, words] int32/uint32 (bit-packed allowed ids), cut [R] int32 (the
    last id that a top-k / top-p cutoff keeps; a column of sample_debug's cut
    will do), first_row [B] int32 (None: sequences follow one another)."""

    __slots__ = ("logits", "temperature", "mask", "cut", "first_row", "V", "device", "c")

    def __init__(self, logits, temperature=None, mask=None, cut=None, first_row=None):
        import torch

        shape, stride, dev, dtype = logits.shape, logits.stride(), logits.device, logits.dtype
        if len(shape) != 2 or (stride[1] != 1 and shape[1] > 1):
            raise ValueError("DistRows: logits must be rows [R, V] with unit inner stride")
        if dtype is not torch.float32 and dtype is not torch.bfloat16:
            raise ValueError("DistRows: logits must be f32 or bf16")
        R, V = shape
        tp = mp = cp = fp = None
        ms = cs = 0
        if temperature is not None:
            if temperature.dtype is not torch.float32 or temperature.device != dev or not temperature.is_contiguous():
                raise ValueError("DistRows: temperature must be contiguous f32 on the logits' device")
            tp = temperature.data_ptr()
        if first_row is not None:
            if first_row.dtype is not torch.int32 or first_row.device != dev or not first_row.is_contiguous():
                raise ValueError("DistRows: first_row must be contiguous int32 on the logits' device")
            fp = first_row.data_ptr()
        if mask is not None:
            if mask.dtype not in (torch.int32, torch.uint32) or mask.device != dev:
                raise ValueError("DistRows: mask must be int32 or uint32 words on the logits' device")
            if mask.dim() != 2 or mask.shape[0] < R or mask.shape[1] * 32 < V or (mask.shape[1] > 1 and mask.stride(1) != 1):
                raise ValueError("DistRows: mask must have a row of words for each logits row")
            mp, ms = mask.data_ptr(), mask.stride(0) if R > 1 else max(mask.stride(0), mask.shape[1])
        if cut is not None:
            if cut.dtype is not torch.int32 or cut.device != dev or cut.dim() != 1 or cut.shape[0] < R:
                raise ValueError("DistRows: cut must have an int32 id for each logits row, on its device")
            cp, cs = cut.data_ptr(), cut.stride(0)
        self.logits, self.temperature, self.mask, self.cut, self.first_row = logits, temperature, mask, cut, first_row
        self.V, self.device = V, dev
        # a single row has no stride to speak of
        self.c = _DistRows(logits.data_ptr(), RL_BF16 if dtype is torch.bfloat16 else RL_F32, R,
                           stride[0] if R > 1 else max(stride[0], V), tp, mp, ms, cp, cs, fp)

    def _of(self, B, who):
        """The C struct, for B sequences."""
        for t in (self.temperature, self.first_row):
            if t is not None and t.numel() != B:
                raise ValueError(f"{who}: temperature and first_row must have an entry for each of {B} sequences")
        return self.c


def _wrong(who, name, t, dtype, shape, dev):
    return ValueError(f"{who}: {name} must be contiguous {dtype} {tuple(shape)} on {dev}, got {t.dtype} {tuple(t.shape)} "
                      f"on {t.device}")


class Q4Weight:
    """4-bit weights with group scales (rl_q4_weight): q [V, H / 2] uint8 packed
    codes, scale [V, H / group] bf16; weight = scale * (code - 8)."""

    __slots__ = ("q", "scale", "group", "V", "H", "device", "c")

    def __init__(self, q, scale, group):
        import torch

        if q.dtype is not torch.uint8 or q.dim() != 2 or (q.shape[1] > 1 and q.stride(1) != 1):
            raise ValueError("Q4Weight: q must be rows of uint8 codes [V, H / 2]")
        if scale.dtype is not torch.bfloat16 or scale.dim() != 2 or (scale.shape[1] > 1 and scale.stride(1) != 1):
            raise ValueError("Q4Weight: scale must be rows of bf16 [V, H / group]")
        V, H = q.shape[0], 2 * q.shape[1]
        if scale.shape[0] != V or scale.shape[1] * group != H or scale.device != q.device:
            raise ValueError(f"Q4Weight: scale {tuple(scale.shape)} on {scale.device} does not fit {V} rows of {H} codes "
                             f"in groups of {group} on {q.device}")
        self.q, self.scale, self.group, self.V, self.H, self.device = q, scale, group, V, H, q.device
        # a single row has no stride to speak of
        self.c = _Q4Weight(q.data_ptr(), q.stride(0) if V > 1 else (H // 2 + 15) // 16 * 16, scale.data_ptr(),
                           scale.stride(0) if V > 1 else H // group, group)


def q4_pack(codes):
    """Codes 0 .. 15 [V, H] as the packed bytes [V, H / 2] of rl_q4_weight."""
    import torch

    V, H = codes.shape
    shifts = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], dtype=torch.int64, device=codes.device)
    word = (codes.to(torch.int64).view(V, H // 8, 8) << shifts).sum(2)
    return torch.where(word >= 1 << 31, word - (1 << 32), word).to(torch.int32).view(torch.uint8)


def q4_unpack(q):
    """The codes 0 .. 15 [V, H] uint8 of packed bytes [V, H / 2]."""
    import torch

    shifts = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], dtype=torch.int32, device=q.device)
    return ((q.contiguous().view(torch.int32)[:, :, None] >> shifts) & 15).flatten(1).to(torch.uint8)


class Sampler:
    """Owns an rl_sampler handle on one device."""

    def __init__(self, device=0, max_batch=256, max_vocab=131072, max_history=1024, flags=0):
        h = ctypes.c_void_p()
        check(lib().rl_sampler_create(ctypes.byref(h), device, max_batch, max_vocab, max_history, flags),
              "rl_sampler_create")
        self.h = h
        self.device = device

    def set_debug(self, flags):
        """rl_sampler_set_debug: RL_DEBUG_* switches (0 = off)."""
        check(lib().rl_sampler_set_debug(self.h, int(flags)), "rl_sampler_set_debug")

    def kernel_times(self):
        """rl_sampler_kernel_times: the last timed call's kernel times (ms)."""
        buf = (ctypes.c_float * 4)()
        n = ctypes.c_int()
        check(lib().rl_sampler_kernel_times(self.h, buf, 4, ctypes.byref(n)), "rl_sampler_kernel_times")
        return [buf[i] for i in range(n.value)]

    def close(self):
        if self.h:
            lib().rl_sampler_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # -- spec profile ---------------------------------------------------------
    def sample(self, logits, params, uniforms, hist=None, hist_len=None, mask=None, out_tok=None,
               out_prob=None, row_status=None, stream=None):
        """logits [B, V] f32/bf16 (cuda), params: torch uint8 view of rl_row_params[B] (cuda)."""
        import torch

        B, V = logits.shape
        dtype = RL_BF16 if logits.dtype == torch.bfloat16 else RL_F32
        dev = logits.device
        if out_tok is None:
            out_tok = torch.empty(B, dtype=torch.int32, device=dev)
        if out_prob is None:
            out_prob = torch.empty(B, dtype=torch.float32, device=dev)
        if row_status is None:
            row_status = torch.empty(B, dtype=torch.int32, device=dev)
        hs = hist.shape[1] if hist is not None else 0
        ms = mask.shape[1] if mask is not None else 0
        check(lib().rl_sample_batch(self.h, _ptr(logits), dtype, B, V, logits.stride(0), _ptr(hist),
                                    _ptr(hist_len), hs, _ptr(mask), ms, _ptr(params), _ptr(uniforms),
                                    _ptr(out_tok), _ptr(out_prob), _ptr(row_status), _stream(stream)),
              "rl_sample_batch")
        return out_tok, out_prob, row_status

    def sample_debug(self, logits, params, uniforms, hist=None, hist_len=None, mask=None, list_cap=1024,
                     stream=None):
        import torch

        B, V = logits.shape
        dtype = RL_BF16 if logits.dtype == torch.bfloat16 else RL_F32
        dev = logits.device
        out_tok = torch.empty(B, dtype=torch.int32, device=dev)
        out_prob = torch.empty(B, dtype=torch.float32, device=dev)
        row_status = torch.empty(B, dtype=torch.int32, device=dev)
        list_ids = torch.full((B, list_cap), -1, dtype=torch.int32, device=dev)
        list_probs = torch.zeros((B, list_cap), dtype=torch.float32, device=dev)
        list_len = torch.zeros(B, dtype=torch.int32, device=dev)
        cut = torch.full((B, 3), -3, dtype=torch.int32, device=dev)
        hs = hist.shape[1] if hist is not None else 0
        ms = mask.shape[1] if mask is not None else 0
        check(lib().rl_sample_batch_debug(self.h, _ptr(logits), dtype, B, V, logits.stride(0), _ptr(hist),
                                          _ptr(hist_len), hs, _ptr(mask), ms, _ptr(params), _ptr(uniforms),
                                          _ptr(out_tok), _ptr(out_prob), _ptr(row_status), _ptr(list_ids),
                                          _ptr(list_probs), _ptr(list_len), list_cap, _ptr(cut), _stream(stream)),
              "rl_sample_batch_debug")
        return out_tok, out_prob, row_status, list_ids, list_probs, list_len, cut

    # -- vocabulary shards -------------------------------------------------------
    def sample_partial(self, logits, vocab_offset, params, hist=None, hist_len=None, mask=None, out_keys=None,
                       out_stats=None, stream=None):
        """One shard's partial result (rl_sample_partial): keys [B, PART_KEYS]
        int64 (the uint64 key bits) and stats [B, 32] uint8 (rl_part_stats)."""
        import torch

        B, V = logits.shape
        dtype = RL_BF16 if logits.dtype == torch.bfloat16 else RL_F32
        dev = logits.device
        if out_keys is None:
            out_keys = torch.empty((B, PART_KEYS), dtype=torch.int64, device=dev)
        if out_stats is None:
            out_stats = torch.empty((B, PART_STATS_DTYPE.itemsize), dtype=torch.uint8, device=dev)
        hs = hist.shape[1] if hist is not None else 0
        ms = mask.shape[1] if mask is not None else 0
        check(lib().rl_sample_partial(self.h, _ptr(logits), dtype, B, V, logits.stride(0), int(vocab_offset),
                                      _ptr(hist), _ptr(hist_len), hs, _ptr(mask), ms, _ptr(params),
                                      _ptr(out_keys), _ptr(out_stats), _stream(stream)),
              "rl_sample_partial")
        return out_keys, out_stats

    def sample_merge(self, keys, stats, params, uniforms, out_tok=None, out_prob=None, row_status=None,
                     stream=None):
        """rl_sample_merge over keys [G, B, PART_KEYS] and stats [G, B, 32]."""
        import torch

        G, B = keys.shape[0], keys.shape[1]
        dev = keys.device
        if out_tok is None:
            out_tok = torch.empty(B, dtype=torch.int32, device=dev)
        if out_prob is None:
            out_prob = torch.empty(B, dtype=torch.float32, device=dev)
        if row_status is None:
            row_status = torch.empty(B, dtype=torch.int32, device=dev)
        check(lib().rl_sample_merge(self.h, G, B, _ptr(keys.contiguous()), _ptr(stats.contiguous()), _ptr(params),
                                    _ptr(uniforms), _ptr(out_tok), _ptr(out_prob), _ptr(row_status),
                                    _stream(stream)),
              "rl_sample_merge")
        return out_tok, out_prob, row_status

    def sample_sharded(self, comm, logits_shard, vocab_offset, V_global, params, uniforms, hist=None, hist_len=None,
                       mask_shard=None, out_tok=None, out_prob=None, row_status=None, stream=None):
        """rl_sample_sharded: this rank's columns [vocab_offset, + width) of
        the rows, one NCCL all-gather on `comm`, the merged draw (global ids).
        The handle needs flags=RL_CREATE_SHARDED."""
        import torch

        B, W = logits_shard.shape
        dtype = RL_BF16 if logits_shard.dtype == torch.bfloat16 else RL_F32
        dev = logits_shard.device
        if out_tok is None:
            out_tok = torch.empty(B, dtype=torch.int32, device=dev)
        if out_prob is None:
            out_prob = torch.empty(B, dtype=torch.float32, device=dev)
        if row_status is None:
            row_status = torch.empty(B, dtype=torch.int32, device=dev)
        hs = hist.shape[1] if hist is not None else 0
        ms = mask_shard.shape[1] if mask_shard is not None else 0
        check(lib().rl_sample_sharded(self.h, ctypes.c_void_p(comm), _ptr(logits_shard), dtype, B, W,
                                      logits_shard.stride(0), int(vocab_offset), int(V_global), _ptr(hist),
                                      _ptr(hist_len), hs, _ptr(mask_shard), ms, _ptr(params), _ptr(uniforms),
                                      _ptr(out_tok), _ptr(out_prob), _ptr(row_status), _stream(stream)),
              "rl_sample_sharded")
        return out_tok, out_prob, row_status

    # -- beam search ----------------------------------------------------------------
    def beam_step(self, logits, items, beams, scores, done, lens=None, alpha=1.0, eos=2, log_softmax=1,
                  n_out=None, stream=None):
        """One BeamSearch::search step for items x beams rows of f32 logits
        (row = item * beams + beam). Returns (beam, tok, score, done), each
        [items, n_out]."""
        import torch

        R, V = logits.shape
        assert R == items * beams
        n_out = 2 * beams if n_out is None else n_out
        dev = logits.device
        ob = torch.empty((items, n_out), dtype=torch.int32, device=dev)
        ot = torch.empty((items, n_out), dtype=torch.int32, device=dev)
        osc = torch.empty((items, n_out), dtype=torch.float32, device=dev)
        od = torch.empty((items, n_out), dtype=torch.uint8, device=dev)
        check(lib().rl_beam_step(self.h, _ptr(logits), items, beams, V, logits.stride(0), _ptr(scores), _ptr(done),
                                 _ptr(lens), float(alpha), int(eos), int(log_softmax), n_out, _ptr(ob), _ptr(ot),
                                 _ptr(osc), _ptr(od), _stream(stream)),
              "rl_beam_step")
        return ob, ot, osc, od

    def sample_host(self, logits, params, uniforms, hist=None, hist_len=None, mask=None):
        """Host numpy buffers in and out (synchronous)."""
        B, V = logits.shape
        out_tok = np.empty(B, np.int32)
        out_prob = np.empty(B, np.float32)
        hs = hist.shape[1] if hist is not None else 0
        ms = mask.shape[1] if mask is not None else 0
        check(lib().rl_sample_host(self.h, _ptr(np.ascontiguousarray(logits, np.float32)), B, V, _ptr(hist),
                                   _ptr(hist_len), hs, _ptr(mask), ms, _ptr(params), _ptr(uniforms),
                                   _ptr(out_tok), _ptr(out_prob)),
              "rl_sample_host")
        return out_tok, out_prob

    def decoder_sample(self, logits, temperature, top_p, uniforms, out_tok=None, out_prob=None, stream=None):
        """rl_decoder_sample: Decoder::sample_with_params semantics on device rows
        [B, V] f32; temperature / top_p / uniforms are [B] f32 device tensors."""
        import torch

        B, V = logits.shape
        dev = logits.device
        if out_tok is None:
            out_tok = torch.empty(B, dtype=torch.int32, device=dev)
        if out_prob is None:
            out_prob = torch.empty(B, dtype=torch.float32, device=dev)
        check(lib().rl_decoder_sample(self.h, _ptr(logits), B, V, logits.stride(0), _ptr(temperature), _ptr(top_p),
                                      _ptr(uniforms), _ptr(out_tok), _ptr(out_prob), _stream(stream)),
              "rl_decoder_sample")
        return out_tok, out_prob

    def decoder_sample_host(self, logits, temperature, top_p, uniforms):
        """rl_decoder_sample_host: Decoder::sample_with_params semantics on host
        rows [B, V] f32 with per-row temperature / top_p / uniform; returns
        (tokens, probs) as numpy arrays."""
        lg = np.ascontiguousarray(logits, np.float32)
        if lg.ndim == 1:
            lg = lg[None, :]
        B, V = lg.shape
        t = np.ascontiguousarray(np.broadcast_to(np.asarray(temperature, np.float32), (B,)))
        p = np.ascontiguousarray(np.broadcast_to(np.asarray(top_p, np.float32), (B,)))
        u = np.ascontiguousarray(np.broadcast_to(np.asarray(uniforms, np.float32), (B,)))
        tok = np.empty(B, np.int32)
        prob = np.empty(B, np.float32)
        check(lib().rl_decoder_sample_host(self.h, _ptr(lg), B, V, _ptr(t), _ptr(p), _ptr(u), _ptr(tok), _ptr(prob)),
              "rl_decoder_sample_host")
        return tok, prob

    def greedy_host(self, logits):
        """rl_greedy_host: argmax (last maximum on ties) of host rows."""
        lg = np.ascontiguousarray(logits, np.float32)
        if lg.ndim == 1:
            lg = lg[None, :]
        tok = np.empty(lg.shape[0], np.int32)
        check(lib().rl_greedy_host(self.h, _ptr(lg), lg.shape[0], lg.shape[1], _ptr(tok)), "rl_greedy_host")
        return tok

    def grammar_greedy_host(self, logits, mask):
        """rl_grammar_greedy_host: argmax over the allowed ids of the bit-packed
        mask rows (lowest id on ties; an all-zero row allows every id)."""
        lg = np.ascontiguousarray(logits, np.float32)
        m = np.ascontiguousarray(mask, np.uint32)
        if lg.ndim == 1:
            lg, m = lg[None, :], m[None, :]
        tok = np.empty(lg.shape[0], np.int32)
        check(lib().rl_grammar_greedy_host(self.h, _ptr(lg), lg.shape[0], lg.shape[1], _ptr(m), m.shape[1], _ptr(tok)),
              "rl_grammar_greedy_host")
        return tok

    def _on_device(self, who, dev):
        """Refuses tensors that are not on the handle's device."""
        if dev.type != "cuda" or dev.index != self.device:
            raise ValueError(f"{who}: the tensors are on {dev}, the sampler on another device")

    # -- speculative decoding ---------------------------------------------------
    def specdec_sample(self, logits, temperature, offset, uniforms, stream=None):
        """rl_specdec_sample: SpeculativeDecoder::sample per row of device
        logits [B, V] f32; temperature / offset / uniforms are [B] device tensors."""
        import torch

        B, V = logits.shape
        out = torch.empty(B, dtype=torch.int32, device=logits.device)
        check(lib().rl_specdec_sample(self.h, _ptr(logits), B, V, logits.stride(0), _ptr(temperature), _ptr(offset),
                                      _ptr(uniforms), _ptr(out), _stream(stream)),
              "rl_specdec_sample")
        return out

    def specdec_verify(self, logits, drafts, n_draft, accept_u, room, draw_u, stream=None):
        """rl_specdec_verify: SpeculativeDecoder::verify_and_accept per request;
        drafts / accept_u [B, Dmax] (same row stride), n_draft / room / draw_u
        [B] (device). Returns (accepted [B], token [B]) device tensors."""
        import torch

        B, V = logits.shape
        if accept_u.stride(0) != drafts.stride(0):
            raise ValueError("specdec_verify: drafts and accept_u need the same row stride")
        dev = logits.device
        acc = torch.empty(B, dtype=torch.int32, device=dev)
        tok = torch.empty(B, dtype=torch.int32, device=dev)
        check(lib().rl_specdec_verify(self.h, _ptr(logits), B, V, logits.stride(0), _ptr(drafts), drafts.stride(0),
                                      _ptr(n_draft), _ptr(accept_u), _ptr(room), _ptr(draw_u), _ptr(acc), _ptr(tok),
                                      _stream(stream)),
              "rl_specdec_verify")
        return acc, tok

    def specdec_verify_draft(self, target, drafts, n_draft, accept_u, draw_u, draft=None, stream=None):
        """rl_specdec_verify_draft: drafts [B, K] int32 (n_draft [B] of them
        valid) against target rows (DistRows, K + 1 a sequence) and the draft
        rows they were drawn from (DistRows, K a sequence; None: given
        drafts); accept_u [B, K] and draw_u [B] f32. Returns (accepted [B],
        tokens [B, K + 1], probs [B, K + 1], row_status [B])."""
        import torch

        who, dev, V = "specdec_verify_draft", target.device, target.V
        i32, f32 = torch.int32, torch.float32
        B, K = shape = drafts.shape
        one = (B,)
        if drafts.dtype is not i32 or drafts.device != dev or not drafts.is_contiguous():
            raise _wrong(who, "drafts", drafts, i32, shape, dev)
        if n_draft.dtype is not i32 or n_draft.shape != one or n_draft.device != dev or not n_draft.is_contiguous():
            raise _wrong(who, "n_draft", n_draft, i32, one, dev)
        if accept_u.dtype is not f32 or accept_u.shape != shape or accept_u.device != dev or not accept_u.is_contiguous():
            raise _wrong(who, "accept_u", accept_u, f32, shape, dev)
        if draw_u.dtype is not f32 or draw_u.shape != one or draw_u.device != dev or not draw_u.is_contiguous():
            raise _wrong(who, "draw_u", draw_u, f32, one, dev)
        if draft is not None and (draft.V != V or draft.device != dev):
            raise ValueError(f"{who}: the draft rows differ from the target rows in V or device")
        self._on_device(who, dev)
        t, d = target._of(B, who), draft._of(B, who) if draft is not None else None
        acc, st = torch.empty_like(n_draft), torch.empty_like(n_draft)
        tok, prob = drafts.new_empty((B, K + 1)), accept_u.new_empty((B, K + 1))
        check(lib().rl_specdec_verify_draft(self.h, B, V, K, t, d, drafts.data_ptr(), n_draft.data_ptr(),
                                            accept_u.data_ptr(), draw_u.data_ptr(), acc.data_ptr(), tok.data_ptr(),
                                            prob.data_ptr(), st.data_ptr(), _raw_stream(stream, dev)),
              "rl_specdec_verify_draft")
        return acc, tok, prob, st

    def specdec_verify_tree(self, target, tokens, parent, n_node, accept_u, draw_u, draft=None, stream=None):
        """rl_specdec_verify_tree: trees of N nodes (tokens, parent [B, N]
        int32, node 0 the root; n_node [B] of them valid) against target rows
        (DistRows, N a sequence) and the draft rows the nodes' children were
        drawn from (DistRows, N a sequence; None: given tokens); accept_u
        [B, N] and draw_u [B] f32. Returns (accepted [B], path [B, N], tokens
        [B, N], probs [B, N], row_status [B])."""
        import torch

        who, dev, V = "specdec_verify_tree", target.device, target.V
        i32, f32 = torch.int32, torch.float32
        B, N = shape = tokens.shape
        one = (B,)
        if tokens.dtype is not i32 or tokens.device != dev or not tokens.is_contiguous():
            raise _wrong(who, "tokens", tokens, i32, shape, dev)
        if parent.dtype is not i32 or parent.shape != shape or parent.device != dev or not parent.is_contiguous():
            raise _wrong(who, "parent", parent, i32, shape, dev)
        if n_node.dtype is not i32 or n_node.shape != one or n_node.device != dev or not n_node.is_contiguous():
            raise _wrong(who, "n_node", n_node, i32, one, dev)
        if accept_u.dtype is not f32 or accept_u.shape != shape or accept_u.device != dev or not accept_u.is_contiguous():
            raise _wrong(who, "accept_u", accept_u, f32, shape, dev)
        if draw_u.dtype is not f32 or draw_u.shape != one or draw_u.device != dev or not draw_u.is_contiguous():
            raise _wrong(who, "draw_u", draw_u, f32, one, dev)
        if draft is not None and (draft.V != V or draft.device != dev):
            raise ValueError(f"{who}: the draft rows differ from the target rows in V or device")
        self._on_device(who, dev)
        t, d = target._of(B, who), draft._of(B, who) if draft is not None else None
        acc, st = torch.empty_like(n_node), torch.empty_like(n_node)
        path, tok, prob = torch.empty_like(tokens), torch.empty_like(tokens), torch.empty_like(accept_u)
        check(lib().rl_specdec_verify_tree(self.h, B, V, N, t, d, tokens.data_ptr(), parent.data_ptr(), n_node.data_ptr(),
                                           accept_u.data_ptr(), draw_u.data_ptr(), acc.data_ptr(), path.data_ptr(),
                                           tok.data_ptr(), prob.data_ptr(), st.data_ptr(), _raw_stream(stream, dev)),
              "rl_specdec_verify_tree")
        return acc, path, tok, prob, st

    # -- LM head ------------------------------------------------------------
    @staticmethod
    def _lm_operands(hidden, weight):
        import torch

        if hidden.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
            raise ValueError("lmhead: hidden and weight must be bf16")
        if hidden.stride(1) != 1 or weight.stride(1) != 1:
            raise ValueError("lmhead: hidden and weight must be row-major (unit inner stride)")
        B, H = hidden.shape
        V, H2 = weight.shape
        if H != H2:
            raise ValueError(f"lmhead: hidden has {H} columns, weight {H2}")
        return B, H, V

    def lmhead_logits(self, hidden, weight, out=None, out_dtype=None, stream=None):
        """rl_lmhead_logits: hidden [B, H] @ weight[V, H]^T on the tensor
        cores (bf16 operands, f32 sums) into out [B, V] (f32 or bf16)."""
        import torch

        B, H, V = self._lm_operands(hidden, weight)
        if out is None:
            out = torch.empty(B, V, dtype=out_dtype or torch.float32, device=hidden.device)
        dt = RL_BF16 if out.dtype == torch.bfloat16 else RL_F32
        check(lib().rl_lmhead_logits(self.h, _ptr(hidden), hidden.stride(0), _ptr(weight), weight.stride(0), B, H, V,
                                     _ptr(out), dt, out.stride(0), _stream(stream)),
              "rl_lmhead_logits")
        return out

    def lmhead_greedy(self, hidden, weight, out_logits=None, stream=None):
        """rl_lmhead_greedy: the last-maximum argmax of each row's logits,
        fused into the GEMM. Returns (tokens [B], row_status [B]); out_logits
        (f32 [B, V], optional) also receives the logits."""
        import torch

        B, H, V = self._lm_operands(hidden, weight)
        tok = torch.empty(B, dtype=torch.int32, device=hidden.device)
        st = torch.empty(B, dtype=torch.int32, device=hidden.device)
        ldo = out_logits.stride(0) if out_logits is not None else V
        check(lib().rl_lmhead_greedy(self.h, _ptr(hidden), hidden.stride(0), _ptr(weight), weight.stride(0), B, H, V,
                                     _ptr(tok), _ptr(st), _ptr(out_logits), ldo, _stream(stream)),
              "rl_lmhead_greedy")
        return tok, st

    def lmhead_sample(self, hidden, weight, params, uniforms, hist=None, hist_len=None, out_tok=None, out_prob=None,
                      row_status=None, stream=None):
        """rl_lmhead_sample: the LM head's logits sampled by the batched
        sampler (same params / uniforms / history as sample())."""
        import torch

        B, H, V = self._lm_operands(hidden, weight)
        dev = hidden.device
        out_tok = out_tok if out_tok is not None else torch.empty(B, dtype=torch.int32, device=dev)
        out_prob = out_prob if out_prob is not None else torch.empty(B, dtype=torch.float32, device=dev)
        row_status = row_status if row_status is not None else torch.empty(B, dtype=torch.int32, device=dev)
        hs = hist.shape[1] if hist is not None else 0
        check(lib().rl_lmhead_sample(self.h, _ptr(hidden), hidden.stride(0), _ptr(weight), weight.stride(0), B, H, V,
                                     _ptr(hist), _ptr(hist_len), hs, _ptr(params), _ptr(uniforms), _ptr(out_tok),
                                     _ptr(out_prob), _ptr(row_status), _stream(stream)),
              "rl_lmhead_sample")
        return out_tok, out_prob, row_status

    # -- LM head, 4-bit weights ------------------------------------------------
    def lmhead_q4_quantize(self, weight, group=128, stream=None):
        """rl_lmhead_q4_quantize: a bf16 weight [V, H] as a Q4Weight."""
        import torch

        if weight.dtype is not torch.bfloat16 or weight.dim() != 2 or weight.stride(1) != 1:
            raise ValueError("lmhead_q4_quantize: weight must be row-major bf16 [V, H]")
        V, H = weight.shape
        if group not in (32, 64, 128) or H % 64 or H % group:
            raise ValueError("lmhead_q4_quantize: group must be 32, 64 or 128, H a multiple of it and of 64")
        dev = weight.device
        self._on_device("lmhead_q4_quantize", dev)
        q = torch.empty(V, H // 2, dtype=torch.uint8, device=dev)
        scale = torch.empty(V, H // group, dtype=torch.bfloat16, device=dev)
        w = Q4Weight(q, scale, group)
        check(lib().rl_lmhead_q4_quantize(self.h, weight.data_ptr(), weight.stride(0) if V > 1 else max(weight.stride(0), H), H, V,
                                          group, w.c.q, w.c.ldq, w.c.scale, w.c.lds, _raw_stream(stream, dev)),
              "rl_lmhead_q4_quantize")
        return w

    def _q4_operands(self, hidden, weight):
        import torch

        if hidden.dtype is not torch.bfloat16 or hidden.dim() != 2 or hidden.stride(1) != 1:
            raise ValueError("lmhead_q4: hidden must be row-major bf16 [B, H]")
        B, H = hidden.shape
        if H != weight.H or hidden.device != weight.device:
            raise ValueError(f"lmhead_q4: hidden has {H} columns on {hidden.device}, weight {weight.H} on {weight.device}")
        self._on_device("lmhead_q4", hidden.device)
        return B, H, hidden.stride(0) if B > 1 else max(hidden.stride(0), H)

    @staticmethod
    def _q4_out(out, B, V, dev, dtypes):
        if out.dtype not in dtypes or out.shape != (B, V) or out.device != dev or (V > 1 and out.stride(1) != 1):
            raise ValueError(f"lmhead_q4: out must be row-major {dtypes} [{B}, {V}] on {dev}")
        return out.stride(0) if B > 1 else max(out.stride(0), V)

    def lmhead_q4_logits(self, hidden, weight, out=None, out_dtype=None, stream=None):
        """rl_lmhead_q4_logits: hidden [B, H] bf16 times a Q4Weight [V, H] into
        out [B, V] (f32 or bf16)."""
        import torch

        B, H, ldh = self._q4_operands(hidden, weight)
        V, dev = weight.V, hidden.device
        if out is None:
            out = torch.empty((B, V), dtype=out_dtype or torch.float32, device=dev)
        ldo = self._q4_out(out, B, V, dev, (torch.float32, torch.bfloat16))
        check(lib().rl_lmhead_q4_logits(self.h, hidden.data_ptr(), ldh, weight.c, B, H, V, out.data_ptr(),
                                        RL_BF16 if out.dtype is torch.bfloat16 else RL_F32, ldo, _raw_stream(stream, dev)),
              "rl_lmhead_q4_logits")
        return out

    def lmhead_q4_greedy(self, hidden, weight, out_logits=None, stream=None):
        """rl_lmhead_q4_greedy: the last-maximum argmax of each row's logits.
        Returns (tokens [B], row_status [B]); out_logits (f32 [B, V],
        optional) also receives the logits."""
        import torch

        B, H, ldh = self._q4_operands(hidden, weight)
        V, dev = weight.V, hidden.device
        tok = torch.empty(B, dtype=torch.int32, device=dev)
        st = torch.empty_like(tok)
        ldo = self._q4_out(out_logits, B, V, dev, (torch.float32,)) if out_logits is not None else V
        check(lib().rl_lmhead_q4_greedy(self.h, hidden.data_ptr(), ldh, weight.c, B, H, V, tok.data_ptr(), st.data_ptr(),
                                        out_logits.data_ptr() if out_logits is not None else None, ldo,
                                        _raw_stream(stream, dev)),
              "rl_lmhead_q4_greedy")
        return tok, st

    def lmhead_q4_sample(self, hidden, weight, params, uniforms, hist=None, hist_len=None, stream=None):
        """rl_lmhead_q4_sample: the 4-bit LM head's logits sampled by the batched
        sampler (same params / uniforms / history as sample()). Returns
        (tokens, probs, row_status)."""
        import torch

        B, H, ldh = self._q4_operands(hidden, weight)
        dev = hidden.device
        tok = torch.empty(B, dtype=torch.int32, device=dev)
        prob = torch.empty(B, dtype=torch.float32, device=dev)
        st = torch.empty_like(tok)
        hs = hist.shape[1] if hist is not None else 0
        check(lib().rl_lmhead_q4_sample(self.h, hidden.data_ptr(), ldh, weight.c, B, H, weight.V, _ptr(hist), _ptr(hist_len),
                                        hs, _ptr(params), _ptr(uniforms), tok.data_ptr(), prob.data_ptr(), st.data_ptr(),
                                        _raw_stream(stream, dev)),
              "rl_lmhead_q4_sample")
        return tok, prob, st

    def sample_host_ptrs(self, logits_p, B, V, params_p, u_p, tok_p, prob_p, hist_p=None, hist_len_p=None,
                         hist_stride=0, mask_p=None, mask_stride=0):
        """Host-pointer variant (pinned buffers) used by the end-to-end benchmark."""
        check(lib().rl_sample_host(self.h, logits_p, B, V, hist_p, hist_len_p, hist_stride, mask_p,
                                   mask_stride, params_p, u_p, tok_p, prob_p),
              "rl_sample_host")


def params_tensor(p: np.ndarray, device):
    """rl_row_params[B] (numpy structured) -> cuda uint8 tensor holding the same bytes."""
    import torch

    return torch.from_numpy(np.ascontiguousarray(p).view(np.uint8).copy()).to(device)


def sample_static(logits, params, uniforms, hist=None, hist_len=None, mask=None, out_tok=None, out_prob=None,
                  row_status=None, stream=None):
    """rl_sample_batch_static: spec sampling on the current device with no
    handle and no allocation inside the call (outputs are allocated here when
    not given). Same arguments and results as Sampler.sample."""
    import torch

    B, V = logits.shape
    dtype = RL_BF16 if logits.dtype == torch.bfloat16 else RL_F32
    dev = logits.device
    if out_tok is None:
        out_tok = torch.empty(B, dtype=torch.int32, device=dev)
    if out_prob is None:
        out_prob = torch.empty(B, dtype=torch.float32, device=dev)
    if row_status is None:
        row_status = torch.empty(B, dtype=torch.int32, device=dev)
    hs = hist.shape[1] if hist is not None else 0
    ms = mask.shape[1] if mask is not None else 0
    # the entry point runs on the current device with that device's scratch:
    # make the tensors' device current, and use its stream
    with torch.cuda.device(dev):
        if stream is None:
            stream = torch.cuda.current_stream(dev)
        _call_static(logits, dtype, B, V, hist, hist_len, hs, mask, ms, params, uniforms, out_tok, out_prob,
                     row_status, stream)
    return out_tok, out_prob, row_status


def _call_static(logits, dtype, B, V, hist, hist_len, hs, mask, ms, params, uniforms, out_tok, out_prob, row_status,
                 stream):
    check(lib().rl_sample_batch_static(_ptr(logits), dtype, B, V, logits.stride(0), _ptr(hist), _ptr(hist_len), hs,
                                       _ptr(mask), ms, _ptr(params), _ptr(uniforms), _ptr(out_tok), _ptr(out_prob),
                                       _ptr(row_status), _stream(stream)),
          "rl_sample_batch_static")


def selfcheck_div(a, T, stream=None):
    """rl_selfcheck_div over device float32 tensors a [n] and T [nT]: per T the
    count of quotients that differ in any bit from IEEE division, and whether
    the fixed-divisor path is in use for it. Returns two cpu numpy arrays."""
    import torch

    nT = T.numel()
    mism = torch.zeros(nT, dtype=torch.int32, device=a.device)
    fast = torch.zeros(nT, dtype=torch.int32, device=a.device)
    check(lib().rl_selfcheck_div(_ptr(a), a.numel(), _ptr(T), nT, _ptr(mism), _ptr(fast), _stream(stream)),
          "rl_selfcheck_div")
    torch.cuda.synchronize(a.device)
    return mism.cpu().numpy().astype(np.uint32), fast.cpu().numpy()


def nccl_unique_id() -> bytes:
    """rl_nccl_unique_id: a new NCCL communicator id (made on one rank)."""
    buf = ctypes.create_string_buffer(NCCL_ID_BYTES)
    check(lib().rl_nccl_unique_id(ctypes.cast(buf, ctypes.c_void_p)), "rl_nccl_unique_id")
    return buf.raw


def nccl_comm_init(nranks: int, id_bytes: bytes, rank: int) -> int:
    """rl_nccl_comm_init on the current device: returns the ncclComm_t as an int."""
    if len(id_bytes) != NCCL_ID_BYTES:
        raise ValueError("an NCCL id has 128 bytes")
    buf = ctypes.create_string_buffer(bytes(id_bytes), NCCL_ID_BYTES)
    c = ctypes.c_void_p()
    check(lib().rl_nccl_comm_init(ctypes.byref(c), int(nranks), ctypes.cast(buf, ctypes.c_void_p), int(rank)),
          "rl_nccl_comm_init")
    return c.value


def nccl_comm_destroy(comm: int) -> None:
    check(lib().rl_nccl_comm_destroy(ctypes.c_void_p(comm)), "rl_nccl_comm_destroy")
