"""Python binding of libtc_hip.so (the C-ABI in include/tc_qmatmul.h, tc_gguf.h,
tc_attention.h and tc_step.h).

The library is the product; this module only passes device pointers, sizes
and the current HIP stream through ctypes, and raises when a call fails.
PyTorch supplies device memory and streams. There is no CPU fallback: if the
library is missing or a call is refused, the call raises.
"""
import ctypes
import os
import struct

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libtc_hip.so")

Q8_0, Q2_K, Q3_K, Q4_K, Q5_K, Q6_K, IQ2_XS, IQ3_XXS, IQ3_S, IQ2_S, IQ4_XS, IQ4_NL, Q5_0 = 8, 10, 11, 12, 13, 14, 17, 18, 21, 22, 23, 20, 6
TYPES = {"Q8_0": Q8_0, "Q2_K": Q2_K, "Q3_K": Q3_K, "Q4_K": Q4_K, "Q5_K": Q5_K, "Q6_K": Q6_K, "IQ3_XXS": IQ3_XXS, "IQ3_S": IQ3_S, "IQ2_S": IQ2_S, "IQ2_XS": IQ2_XS, "IQ4_XS": IQ4_XS, "IQ4_NL": IQ4_NL, "Q5_0": Q5_0}
TYPE_SIZE = {Q8_0: 34, Q2_K: 84, Q3_K: 110, Q4_K: 144, Q5_K: 176, Q6_K: 210, IQ3_XXS: 98, IQ3_S: 110, IQ2_S: 82, IQ2_XS: 74, IQ4_XS: 136, IQ4_NL: 18, Q5_0: 22}
BLOCK_SIZE = {Q8_0: 32, Q2_K: 256, Q3_K: 256, Q4_K: 256, Q5_K: 256, Q6_K: 256, IQ3_XXS: 256, IQ3_S: 256, IQ2_S: 256, IQ2_XS: 256, IQ4_XS: 256, IQ4_NL: 32, Q5_0: 32}

TC_OK, TC_E_UNSUPPORTED, TC_E_LAUNCH, TC_E_ARG = 0, -1, -2, -3

# Element types of rows and caches (tc_attention.h).
F32, F16, I8, BF16, E4M3 = 0, 1, 24, 30, 100

# Every function the C headers declare, with its ctypes signature.
_P, _U32, _I = ctypes.c_void_p, ctypes.c_uint32, ctypes.c_int
SIGNATURES = {
    "tc_available": (_I, []),
    "tc_gemv": (_I, [_I, _P, _P, _P, _U32, _U32, _U32, _P]),
    "tc_gemv_reserve": (_I, [_U32, _U32]),
    "tc_gemv_multi": (_I, [_I, _U32, _P, _P, _P, _P, _P, _U32, _P]),
    "tc_act_bytes": (ctypes.c_size_t, [_I, _U32, _U32]),
    "tc_act_quantize": (_I, [_I, _P, _U32, _U32, _P, _P]),
    "tc_gemv_q8": (_I, [_I, _P, _P, _P, _U32, _U32, _U32, _P]),
    "tc_gemv_dual": (_I, [_I, _P, _P, _P, _P, _P, _U32, _U32, _P]),
    "tc_gemm": (_I, [_I, _P, _P, _P, _U32, _U32, _U32, _U32, _P]),
    "tc_gemm_preferred": (_I, [_U32, _U32, _U32]),
    "tc_gemm_set_q8_enabled": (None, [_I]),
    "tc_quantize_act": (_I, [_I, _P, _U32, _U32, _P, _P, _P, _P]),
    "tc_block_isums": (_I, [_I, _P, _P, _P, _U32, _U32, _U32, _P]),
    "tc_encode": (_I, [_I, _P, _P, _U32, _U32, _P]),
    "tc_row_bytes": (ctypes.c_size_t, [_I, _U32]),
    "tc_moe_ffn": (_I, [_P, _P, _P, _U32, _U32, _P, _P, _P, _U32, _U32, _U32, _P, _P]),
    "tc_debug_q8k_row": (_I, [_I, _P, _U32, _P, _U32, _P]),
    "tc_debug_q8_0_row": (_I, [_P, _U32, _P, _U32, _P]),
    "tc_debug_q8k_blocks": (_I, [_I, _P, _U32, _P, _U32, _P, _P]),
    "tc_debug_q8_0_blocks": (_I, [_P, _U32, _P, _U32, _P, _P]),
    "tc_last_error": (ctypes.c_char_p, []),
    "tc_probe_sink_bytes": (ctypes.c_size_t, []),
    "tc_probe_mfma_i8": (_I, [_U32, _U32, _P, _P]),
    "tc_probe_read": (_I, [_P, ctypes.c_size_t, _U32, _P, _P]),
    "tc_moe_set_gemm_min_tokens": (None, [_U32]),
    "tc_moe_router": (_I, [_P, _P, _U32, _U32, _U32, _U32, _P, _P, _P, _P]),
    "tc_moe_select": (_I, [_P, _U32, _U32, _U32, _P, _P, _P]),
    "tc_host_matmul": (_I, [_I, _P, _P, _U32, _U32, _U32, _P, _P]),
    "tc_host_matmul_f32": (_I, [_P, _P, _U32, _U32, _U32, _P]),
    "tc_gemm_noalloc": (_I, [_I, _P, _P, _P, _U32, _U32, _U32, _U32, _P]),
    "tc_gemm_noalloc_scratch_bytes": (ctypes.c_size_t, []),
    "tc_host_weights_register": (_I, [_P, ctypes.c_size_t]),
    "tc_host_weights_unregister": (_I, [_P]),
    "tc_kv_write": (_I, [_P, _P, _I, _P, _P, _U32, _U32, _P]),
    "tc_kv_read": (_I, [_P, _P, _I, _P, _P, _P]),
    "tc_attn": (_I, [_P, _P, _I, _P, _U32, _P, _U32, ctypes.c_float, _U32, _P]),
    "tc_attn_reserve": (_I, [_U32, _U32]),
    "tc_spec_verify": (_I, [_P, _P, _U32, _U32, _U32, _P, _P, _P, _P, _P, _P, _P, _P]),
    "tc_kv_plan": (_I, [_P, _P]),
    "tc_norm_add": (_I, [_P, _P]),
    "tc_rope_turns": (_I, [_P, _U32, ctypes.c_double, _P, _P, _P]),
    "tc_rope_apply": (_I, [_P, _I, _P, _U32, _P, _U32, _P, _U32, _U32, _U32, _P]),
    "tc_rope_kv_write": (_I, [_P, _P, _P, _I, _P, _U32, _P, _U32, _P, _U32, _P, _U32, _P, _P, ctypes.c_float, _P]),
    "tc_logits_adjust": (_I, [_P, _I, _P, _U32, _U32, _U32, _U32, _P, _P, _P, _U32, _P]),
    "tc_gguf_open": (_P, [ctypes.c_char_p]),
    "tc_gguf_open_metadata": (_P, [ctypes.c_char_p]),
    "tc_gguf_close": (None, [_P]),
    "tc_gguf_version": (_U32, [_P]),
    "tc_gguf_tensor_count": (ctypes.c_uint64, [_P]),
    "tc_gguf_metadata_count": (ctypes.c_uint64, [_P]),
    "tc_gguf_data_offset": (ctypes.c_uint64, [_P]),
    "tc_gguf_find_tensor": (ctypes.c_int64, [_P, ctypes.c_char_p]),
    "tc_gguf_tensor_info": (_I, [_P, ctypes.c_uint64, ctypes.POINTER(ctypes.c_char_p), ctypes.POINTER(_U32),
                                 ctypes.POINTER(_U32), ctypes.POINTER(ctypes.c_uint64),
                                 ctypes.POINTER(ctypes.c_uint64), ctypes.POINTER(ctypes.c_uint64)]),
    "tc_gguf_tensor_data": (_P, [_P, ctypes.c_uint64]),
    "tc_gguf_upload": (_I, [_P, ctypes.c_uint64, _P, ctypes.c_uint64, _P]),
    "tc_gguf_meta": (ctypes.c_char_p, [_P, ctypes.c_char_p]),
    "tc_gguf_type_size": (_U32, [_U32]),
    "tc_gguf_block_size": (_U32, [_U32]),
}


class TCError(RuntimeError):
    def __init__(self, code, msg):
        super().__init__(f"libtc_hip error {code}: {msg}")
        self.code = code


def row_bytes(qtype, cols):
    return cols // BLOCK_SIZE[qtype] * TYPE_SIZE[qtype]


_LOADED = {}


def load_library(path=LIB_PATH):
    if path in _LOADED:
        return _LOADED[path]
    # torch ships its own libamdhip64.so.7; it must be the HIP runtime this
    # library binds to, or the streams and memory torch hands over belong to
    # another runtime instance. Importing torch first makes the loader reuse it.
    import torch  # noqa: F401
    if not os.path.exists(path):
        raise FileNotFoundError(f"{path} is not built: run __graft_entry__.build() "
                                "(make -C tinycoder-inference_amd)")
    lib = ctypes.CDLL(path)
    for name, (res, args) in SIGNATURES.items():
        f = getattr(lib, name)
        f.restype = res
        f.argtypes = args
    _elem_types()
    _LOADED[path] = lib
    return lib


_ELEM_TYPES = {}


def _elem_types():
    if not _ELEM_TYPES:
        import torch
        _ELEM_TYPES.update({torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16, torch.int8: I8,
                            torch.float8_e4m3fn: E4M3})
    return _ELEM_TYPES


def _elem_type(dtype):
    """The tc_attention.h element type of a torch dtype."""
    t = _elem_types().get(dtype)
    if t is None:
        raise TCError(TC_E_UNSUPPORTED, f"no element type for {dtype}")
    return t


class _CKVCache(ctypes.Structure):
    _fields_ = [("type", ctypes.c_int32), ("n_pages", _U32), ("kv_heads", _U32), ("page_tokens", _U32),
                ("head_dim", _U32), ("k", _P), ("v", _P), ("k_scale", _P), ("v_scale", _P)]


class _CKVBatch(ctypes.Structure):
    _fields_ = [("n_seq", _U32), ("n_tokens", _U32), ("table_pages", _U32), ("start", _P), ("len", _P), ("table", _P)]


def _need(ok, what):
    if not ok:
        raise TCError(TC_E_ARG, what)


def _u32(x, name):
    """x, which ctypes would cut to 32 bits without a word."""
    if not 0 <= x <= 0xFFFFFFFF:
        raise TCError(TC_E_ARG, f"{name}={x} is not a number of 32 bits")
    return x


class KVCache:
    """The buffers of one layer's paged cache (tc_kv_cache): k and v
    [n_pages][kv_heads][page_tokens][head_dim] of float16, bfloat16, int8 or
    float8_e4m3fn, for the 8-bit types with k_scale and v_scale fp32
    [n_pages][kv_heads][page_tokens]."""

    def __init__(self, k, v, k_scale=None, v_scale=None):
        import torch
        _need(k.dim() == 4 and k.shape == v.shape and k.dtype == v.dtype, "k and v differ or are not 4-dimensional")
        scaled = k.dtype in (torch.int8, torch.float8_e4m3fn)
        for t in (k_scale, v_scale):
            _need((t is not None) == scaled, "scales go with the 8-bit types and with these only")
            _need(t is None or (t.dtype == torch.float32 and t.shape == k.shape[:3]), "scales are fp32 [n_pages][kv_heads][page_tokens]")
        held = [t for t in (k, v, k_scale, v_scale) if t is not None]
        _need(all(t.is_contiguous() and t.device == k.device for t in held), "a cache is contiguous and on one device")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.n_pages, self.kv_heads, self.page_tokens, self.head_dim = k.shape
        self.device = k.get_device()  # (-1: the CPU)
        self.c = _CKVCache(_elem_type(k.dtype), self.n_pages, self.kv_heads, self.page_tokens, self.head_dim,
                           *[None if t is None else t.data_ptr() for t in (k, v, k_scale, v_scale)])
        self.ref = ctypes.byref(self.c)

    @classmethod
    def empty(cls, dtype, n_pages, kv_heads, page_tokens, head_dim, device="cuda"):
        """A cache of zeros."""
        import torch
        shape = (n_pages, kv_heads, page_tokens, head_dim)
        k, v = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
        if dtype not in (torch.int8, torch.float8_e4m3fn):
            return cls(k, v)
        return cls(k, v, *(torch.zeros(shape[:3], dtype=torch.float32, device=device) for _ in range(2)))


class KVBatch:
    """Which rows are whose, and where they lie (tc_kv_batch): start int32
    [n_seq + 1], length int32 [n_seq], table int32 [n_seq][table_pages]. Other
    lengths and pages may be written into the tensors between calls."""

    def __init__(self, start, length, table):
        import torch
        n = length.numel()
        _need(all(t.dtype == torch.int32 and t.is_contiguous() and t.device == start.device for t in (start, length, table)),
              "start, length and table are contiguous int32 on one device")
        _need(start.numel() == n + 1 and table.dim() == 2 and table.shape[0] == n,
              "start has n_seq + 1 entries, table n_seq rows")
        self.start, self.length, self.table = start, length, table
        self.device = start.get_device()
        self._of = {}  # a struct for each number of rows: calls at once share none that changes

    def of(self, n_tokens):
        """The C struct of a call with n_tokens rows, by reference."""
        ref = self._of.get(n_tokens)
        if ref is None:
            if len(self._of) >= 64:
                self._of.clear()
            c = _CKVBatch(self.length.numel(), n_tokens, self.table.shape[1], self.start.data_ptr(), self.length.data_ptr(),
                          self.table.data_ptr())
            ref = self._of[n_tokens] = ctypes.byref(c)
        return ref


class _CPlan(ctypes.Structure):
    _fields_ = [(n, _U32) for n in ("n_seq", "n_tokens", "page_tokens", "table_pages", "ring_pages")] + \
               [(n, _P) for n in ("new_tokens", "held", "pages", "free", "table", "ring", "start", "len", "pages_out",
                                  "free_out", "sequence", "position", "slot")]


class _CNorm(ctypes.Structure):
    _fields_ = [("kind", ctypes.c_int32), ("eps", ctypes.c_float), ("weight", _P), ("bias", _P), ("offset", ctypes.c_float)]


class _CNormRows(ctypes.Structure):
    _fields_ = [("n_rows", _U32), ("cols", _U32), ("h", _P), ("y", _P), ("h_out", _P), ("x", _P),
                ("h_type", ctypes.c_int32), ("y_type", ctypes.c_int32), ("x_type", ctypes.c_int32),
                ("h_stride", _U32), ("y_stride", _U32), ("h_out_stride", _U32), ("x_stride", _U32),
                ("post", _P), ("pre", _P), ("gate", _P), ("gate_kind", ctypes.c_int32), ("gate_type", ctypes.c_int32),
                ("gate_sigmoid", ctypes.c_int32), ("scale", ctypes.c_float), ("act_type", ctypes.c_int32), ("act", _P)]


# the same by struct.pack (native sizes and alignment, as ctypes')
_PACK_NORM_ROWS = struct.Struct("IIPPPPiiiIIIIPPPiiifiP").pack


class _CRope(ctypes.Structure):
    _fields_ = [("n_rot", _U32), ("layout", ctypes.c_int32), ("turns", _P), ("factor", ctypes.c_float)]


class _CRopeScaling(ctypes.Structure):
    _fields_ = [("kind", ctypes.c_int32)] + [(n, ctypes.c_double) for n in ("factor", "original", "low", "high")] + \
               [("divisors", _P)]


class _CLogitRules(ctypes.Structure):
    _fields_ = [("repetition", _P), ("frequency", _P), ("presence", _P), ("history", _P), ("history_start", _P), ("prompt", _P),
                ("n_history", _U32), ("bias_start", _P), ("bias_token", _P), ("bias_value", _P), ("n_bias", _U32), ("mask", _P),
                ("n_masks", _U32), ("mask_words", _U32), ("mask_of", _P)]


def _same_device(ts, what):
    """The one device index of tensors (or Nones), -1 for the CPU."""
    ts = [t for t in ts if t is not None]
    _need(all(t.is_contiguous() and t.device == ts[0].device for t in ts), what)
    return ts[0].get_device()


class KVPlan:
    """The geometry of a batch's steps (tc_plan): the sequences' state, and what
    Library.kv_plan makes of it. All int32, contiguous, on one device:

      new     [n_seq]   tokens that each sequence brings to the step, -1: it has ended
      held    [n_seq]   tokens it has in the cache
      pages   [n_seq]   pages it has in the table
      table   [n_seq][table_pages]; new pages are entered
      ring    [pages]   pages not in use, free[1] of them from ring[free[0]] on
      free    [2 or 3]

    Behind a call: `batch` (a KVBatch of start, length and table), start [n_seq + 1],
    length, pages_out [n_seq], free_out [3] (its last entry: pages that were missing),
    and of each of n_tokens rows its sequence, position (int32) and slot (int64), -1 behind
    the last sequence. in_place: length, pages_out and free_out are held, pages and free
    (which has 3 entries then), so that the next call goes on from there."""

    def __init__(self, new, held, pages, table, ring, free, page_tokens, n_tokens, in_place=False):
        import torch
        n = new.numel()
        given = (new, held, pages, table, ring, free)
        _need(all(t.dtype == torch.int32 for t in given), "a plan's arrays are int32")
        self.device = _same_device(given, "a plan's arrays are contiguous and on one device")
        _need(held.numel() == pages.numel() == n and table.dim() == 2 and table.shape[0] == n,
              "held and pages have an entry for each sequence, table a row")
        _need(free.numel() == 3 or (free.numel() == 2 and not in_place), "free has 2 entries, or 3")
        self.new, self.held, self.pages, self.table, self.ring, self.free = given

        _u32(n_tokens, "n_tokens")
        self.slot = torch.zeros(n_tokens, dtype=torch.int64, device=new.device)
        sizes = [n + 1, n_tokens, n_tokens] + ([] if in_place else [n, n, 3])
        made = torch.zeros(sum(sizes), dtype=torch.int32, device=new.device).split(sizes)
        self.start, self.sequence, self.position = made[:3]
        self.length, self.pages_out, self.free_out = (held, pages, free) if in_place else made[3:]
        self.n_tokens, self.page_tokens = n_tokens, page_tokens
        self.batch = KVBatch(self.start, self.length, table)
        self.c = _CPlan(n, n_tokens, _u32(page_tokens, "page_tokens"), table.shape[1], ring.numel(),
                        *[t.data_ptr() for t in (new, held, pages, free, table, ring, self.start, self.length, self.pages_out,
                                                 self.free_out, self.sequence, self.position, self.slot)])
        self.ref = ctypes.byref(self.c)


NORM_KINDS = {"rms": 0, "layer": 1}


class Norm:
    """A norm and its weights (tc_norm): fp32 weight and bias [cols], either None;
    offset is added to the weights."""

    def __init__(self, weight=None, bias=None, eps=1e-6, kind="rms", offset=0.0):
        import torch
        _need(kind in NORM_KINDS, f"a norm is one of {sorted(NORM_KINDS)}")
        self.weight, self.bias = weight, bias
        held = [t for t in (weight, bias) if t is not None]
        _need(all(t.dtype == torch.float32 and t.dim() == 1 for t in held), "a norm's weights are fp32 [cols]")
        self.device = _same_device(held, "a norm's weights are contiguous and on one device") if held else None
        _need(len({t.numel() for t in held}) <= 1, "weight and bias differ in size")
        self.cols = held[0].numel() if held else None
        self.c = _CNorm(NORM_KINDS[kind], eps, *[None if t is None else t.data_ptr() for t in (weight, bias)], offset)
        self.ref = ctypes.addressof(self.c)

    def of(self, cols, device):
        """The C struct's address, for rows of `cols` values on a device."""
        if self.cols is not None and (self.cols != cols or self.device != device):
            raise TCError(TC_E_ARG, "a norm's weights are not the rows' or not on the current device")
        return self.ref


ROPE_LAYOUTS = {"half": 0, "pairs": 1}
ROPE_SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3, "bands": 4}


class Rope:
    """Rotary positions of a head's first n_rot dims (tc_rope), with their table of
    frequencies on `device`. layout: "half" (dims i and i + n_rot / 2 are a pair) or
    "pairs" (2i and 2i + 1). scaling: "none", "linear", "ntk", "yarn" or "bands", with the
    numbers of tc_rope_scaling; divisors: fp32 [n_rot / 2]. factor_of_values: instead of the
    scaling's own factor of the rotated values. The table is there when the object is, for any stream; one made
    during a capture is filled when the graph runs."""

    def __init__(self, n_rot, theta=10000.0, layout="half", scaling="none", factor=1.0, original=0.0, low=0.0, high=0.0,
                 divisors=None, factor_of_values=None, device="cuda"):
        import torch
        _need(layout in ROPE_LAYOUTS, f"a layout is one of {sorted(ROPE_LAYOUTS)}")
        _need(scaling in ROPE_SCALINGS, f"a scaling is one of {sorted(ROPE_SCALINGS)}")
        _need(n_rot > 0 and n_rot % 2 == 0, "n_rot is even")
        _need(divisors is None or (divisors.dtype == torch.float32 and divisors.is_contiguous() and divisors.numel() == n_rot // 2),
              "divisors are contiguous fp32 [n_rot / 2]")
        _need(torch.device(device).type == "cuda", "a rope's table is on a GPU")
        lib = load_library()
        self.n_rot, self.layout = n_rot, layout
        self.turns = torch.empty(n_rot // 2, dtype=torch.float64, device=device)
        _need(divisors is None or divisors.device == self.turns.device, "divisors are on the rope's device")
        self.divisors = divisors
        self.device = self.turns.get_device()
        f = ctypes.c_float()
        c = _CRopeScaling(ROPE_SCALINGS[scaling], factor, original, low, high, None if divisors is None else divisors.data_ptr())
        with torch.cuda.device(self.device):
            rc = lib.tc_rope_turns(ctypes.byref(c), n_rot, theta, self.turns.data_ptr(), ctypes.byref(f),
                                   torch.cuda.current_stream().cuda_stream)
            if rc != TC_OK:
                raise TCError(rc, lib.tc_last_error().decode())
            # (made once, used on any stream: the table is there when this returns)
            if not torch.cuda.is_current_stream_capturing():
                torch.cuda.current_stream().synchronize()
        self.c = _CRope(n_rot, ROPE_LAYOUTS[layout], self.turns.data_ptr(), f.value if factor_of_values is None else factor_of_values)
        self.ref = ctypes.byref(self.c)


class LogitRules:
    """What is done to a batch's logits (tc_logit_rules), every tensor contiguous, on one
    device, or None: repetition, frequency, presence fp32 [n_seq]; history int32 (the
    sequences' tokens one behind the other) with history_start int32 [n_seq + 1] and
    prompt int32 [n_seq] (how many of them were asked; -n: n of them and of the step's tokens
    behind them, for prompts among the rows); bias_token int32, bias_value fp32 with bias_start int32
    [n_seq + 1]; mask int32 [n_masks][words] (32 tokens a word) with mask_of int32
    [n_tokens]. Other numbers may be written into the tensors between calls."""

    def __init__(self, repetition=None, frequency=None, presence=None, history=None, history_start=None, prompt=None,
                 bias_start=None, bias_token=None, bias_value=None, mask=None, mask_of=None):
        import torch
        floats, ints = (repetition, frequency, presence, bias_value), (history, history_start, prompt, bias_start, bias_token,
                                                                       mask, mask_of)
        _need(all(t is None or t.dtype == torch.float32 for t in floats), "penalties and biases are fp32")
        _need(all(t is None or t.dtype == torch.int32 for t in ints), "tokens, their places and masks are int32")
        held = [t for t in floats + ints if t is not None]
        self.device = _same_device(held, "rules are contiguous and on one device") if held else None
        _need((history is None) == (history_start is None), "history goes with history_start")
        _need((bias_start is None) == (bias_token is None) == (bias_value is None), "bias_start, bias_token and bias_value go together")
        _need(bias_token is None or bias_token.numel() == bias_value.numel(), "bias_token and bias_value differ in size")
        _need(mask is None or mask.dim() == 2, "a mask is [n_masks][words]")
        _need(mask_of is None or mask is not None, "mask_of without masks")
        _need(prompt is None or history is not None, "prompt without a history")
        self.held = held
        sizes = {t.numel() for t in (repetition, frequency, presence, prompt) if t is not None} | \
                     {t.numel() - 1 for t in (history_start, bias_start) if t is not None}
        _need(len(sizes) <= 1, "the rules are of different numbers of sequences")
        self.n_seq = sizes.pop() if sizes else None
        # rows that mask_of has an entry for
        self.rows = None if mask_of is None else mask_of.numel()
        self.words = None if mask is None else mask.shape[1]
        p = [None if t is None else t.data_ptr() for t in (repetition, frequency, presence, history, history_start, prompt,
                                                           bias_start, bias_token, bias_value, mask, mask_of)]
        self.c = _CLogitRules(*p[:6], 0 if history is None else _u32(history.numel(), "history"), *p[6:9],
                              0 if bias_token is None else _u32(bias_token.numel(), "biases"), p[9],
                              0 if mask is None else _u32(mask.shape[0], "masks"), 0 if mask is None else mask.shape[1], p[10])
        self.ref = ctypes.byref(self.c)


def _ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


class Library:
    """Thin callable wrapper; tensors are torch CUDA tensors."""

    def __init__(self, path=LIB_PATH):
        self.lib = load_library(path)
        self.path = path
        import torch
        self._torch = torch
        self._raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        # (torch.cuda's own look at whether it is initialised takes longer than the rest of it)
        quick = getattr(torch._C, "_cuda_getDevice", None)
        self._current_device = quick if quick is not None and torch.cuda.is_initialized() else torch.cuda.current_device

    # -- helpers ---------------------------------------------------------------
    def _stream(self, device=None):
        # The current device's current stream as a handle: reading it without
        # building a torch.cuda.Stream object takes 0.4 instead of 2.9 us, a
        # quarter of a small call's host time (10.1 -> 7.6 us for tc_gemv).
        raw = self._raw_stream
        if raw is None:
            import torch
            return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        return ctypes.c_void_p(raw(self._current_device() if device is None else device))

    def _check(self, rc):
        if rc != TC_OK:
            raise TCError(rc, self.lib.tc_last_error().decode())
        return rc

    def available(self):
        return bool(self.lib.tc_available())

    # -- entry points -------------------------------------------------------------
    def gemv(self, qtype, w, x, rows, cols, out=None):
        import torch
        S = x.numel() // cols
        if out is None:
            out = torch.empty((S, rows), dtype=torch.float32, device=x.device)
        self._check(self.lib.tc_gemv(qtype, _ptr(w), _ptr(x), _ptr(out), S, rows, cols, self._stream()))
        return out

    def gemv_multi(self, qtype, ws, xs, rows, cols, outs=None):
        """One launch over several matrices; xs[i] is [S][cols[i]]."""
        import torch
        n = len(ws)
        S = xs[0].numel() // cols[0]
        if outs is None:
            outs = [torch.empty((S, rows[i]), dtype=torch.float32, device=xs[0].device) for i in range(n)]
        arr = ctypes.c_void_p * n
        u32 = ctypes.c_uint32 * n
        self._check(self.lib.tc_gemv_multi(qtype, n, arr(*[w.data_ptr() for w in ws]),
                                           arr(*[x.data_ptr() for x in xs]), arr(*[o.data_ptr() for o in outs]),
                                           u32(*rows), u32(*cols), S, self._stream()))
        return outs

    def act_buffer(self, qtype, seq_len, cols, device="cuda"):
        import torch
        n = self.lib.tc_act_bytes(qtype, seq_len, cols)
        if n == 0:
            raise TCError(TC_E_UNSUPPORTED, f"no activation layout for type {qtype}, cols {cols}")
        return torch.empty(n, dtype=torch.uint8, device=device)

    def act_quantize(self, qtype, x, cols, act):
        S = x.numel() // cols
        self._check(self.lib.tc_act_quantize(qtype, _ptr(x), S, cols, _ptr(act), self._stream()))
        return act

    def gemv_q8(self, qtype, w, act, seq_len, rows, cols, out=None):
        import torch
        if out is None:
            out = torch.empty((seq_len, rows), dtype=torch.float32, device=act.device)
        self._check(self.lib.tc_gemv_q8(qtype, _ptr(w), _ptr(act), _ptr(out), seq_len, rows, cols,
                                        self._stream()))
        return out

    def gemm(self, qtype, w, x, rows, cols, out=None):
        import torch
        S = x.numel() // cols
        if out is None:
            out = torch.empty((S, rows), dtype=torch.float32, device=x.device)
        self._check(self.lib.tc_gemm(qtype, _ptr(w), _ptr(x), _ptr(out), S, rows, cols,
                                     cols // BLOCK_SIZE[qtype], self._stream()))
        return out

    def gemv_dual(self, qtype, wg, wu, x, rows, cols):
        import torch
        g = torch.empty(rows, dtype=torch.float32, device=x.device)
        u = torch.empty(rows, dtype=torch.float32, device=x.device)
        self._check(self.lib.tc_gemv_dual(qtype, _ptr(wg), _ptr(wu), _ptr(x), _ptr(g), _ptr(u), rows,
                                          cols, self._stream()))
        return g, u

    def quantize_act(self, qtype, x, cols):
        import torch
        S = x.numel() // cols
        blk = 32 if qtype == Q8_0 else 256
        qs = torch.empty((S, cols), dtype=torch.int8, device=x.device)
        d = torch.empty((S, cols // blk), dtype=torch.float32, device=x.device)
        bs = None if qtype == Q8_0 else torch.empty((S, cols // 16), dtype=torch.int16, device=x.device)
        self._check(self.lib.tc_quantize_act(qtype, _ptr(x), S, cols, _ptr(qs), _ptr(d), _ptr(bs),
                                             self._stream()))
        return qs, d, bs

    def block_isums(self, qtype, w, x, rows, cols):
        import torch
        S = x.numel() // cols
        nb = cols // BLOCK_SIZE[qtype]
        k = 8 if qtype in (Q4_K, Q5_K) else 2 if qtype == Q2_K else 1
        out = torch.empty((S, rows, nb, k), dtype=torch.int32, device=x.device)
        self._check(self.lib.tc_block_isums(qtype, _ptr(w), _ptr(x), _ptr(out), S, rows, cols,
                                            self._stream()))
        return out

    def encode(self, qtype, x):
        import torch
        rows, cols = x.shape
        out = torch.empty(rows * row_bytes(qtype, cols), dtype=torch.uint8, device=x.device)
        self._check(self.lib.tc_encode(qtype, _ptr(x), _ptr(out), rows, cols, self._stream()))
        return out

    def debug_row(self, qtype, w_row, x):
        """Host numpy row + host x -> the decode kernel's row result."""
        import numpy as np
        w_row = np.ascontiguousarray(w_row, np.uint8)
        x = np.ascontiguousarray(x, np.float32).ravel()
        res = np.zeros(1, np.float32)
        cols = x.size
        if qtype == Q8_0:
            self._check(self.lib.tc_debug_q8_0_row(w_row.ctypes.data, cols // 32, x.ctypes.data, cols,
                                                   res.ctypes.data))
        else:
            self._check(self.lib.tc_debug_q8k_row(qtype, w_row.ctypes.data, cols // 256, x.ctypes.data, cols,
                                                  res.ctypes.data))
        return float(res[0])

    def debug_blocks(self, qtype, w_row, x):
        """-> (per-block float contributions, quantized activation block bytes)."""
        import numpy as np
        w_row = np.ascontiguousarray(w_row, np.uint8)
        x = np.ascontiguousarray(x, np.float32).ravel()
        cols = x.size
        if qtype == Q8_0:
            nb = cols // 32
            blk, q = np.zeros(nb, np.float32), np.zeros(nb * 36, np.uint8)
            self._check(self.lib.tc_debug_q8_0_blocks(w_row.ctypes.data, nb, x.ctypes.data, cols, blk.ctypes.data,
                                                      q.ctypes.data))
        else:
            nb = cols // 256
            blk, q = np.zeros(nb, np.float32), np.zeros(nb * 292, np.uint8)
            self._check(self.lib.tc_debug_q8k_blocks(qtype, w_row.ctypes.data, nb, x.ctypes.data, cols,
                                                     blk.ctypes.data, q.ctypes.data))
        return blk, q

    def moe_ffn(self, x, ids, wts, wg, wu, wd, n_experts, hidden, ff, out=None):
        import torch
        S, K = ids.shape
        if out is None:
            out = torch.empty((S, hidden), dtype=torch.float32, device=x.device)
        self._check(self.lib.tc_moe_ffn(_ptr(x), _ptr(ids), _ptr(wts), S, K, _ptr(wg), _ptr(wu), _ptr(wd),
                                        n_experts, hidden, ff, _ptr(out), self._stream()))
        return out

    def moe_router(self, w_router, x, top_k):
        """Router logits, expert ids and weights for x [S][hidden] against the
        fp32 router matrix [n_experts][hidden]."""
        import torch
        E, H = w_router.shape
        S = x.numel() // H
        logits = torch.empty((S, E), dtype=torch.float32, device=x.device)
        ids = torch.empty((S, top_k), dtype=torch.int32, device=x.device)
        wts = torch.empty((S, top_k), dtype=torch.float32, device=x.device)
        self._check(self.lib.tc_moe_router(_ptr(w_router), _ptr(x), S, E, H, top_k, _ptr(logits), _ptr(ids),
                                           _ptr(wts), self._stream()))
        return logits, ids, wts

    def moe_select(self, logits, top_k):
        import torch
        S, E = logits.shape
        ids = torch.empty((S, top_k), dtype=torch.int32, device=logits.device)
        wts = torch.empty((S, top_k), dtype=torch.float32, device=logits.device)
        self._check(self.lib.tc_moe_select(_ptr(logits), S, E, top_k, _ptr(ids), _ptr(wts), self._stream()))
        return ids, wts


    # -- paged cache, attention, drafted tokens ---------------------------------------
    # (a call's host time is a small call's whole time, so its checks cost no more than they must: 10.5 -> 6.9 us
    # for tc_kv_write)
    def _kv_call(self, cache, batch, x, y, strided):
        """Checks of rows x and y [n_tokens][heads][head_dim], of which the first
        `strided` may have strides; -> n_tokens, current stream."""
        import torch
        shape = x.shape
        if len(shape) != 3 or y.shape != shape or y.dtype != x.dtype:
            raise TCError(TC_E_ARG, "rows are [n_tokens][heads][head_dim], of one type")
        T, H, D = shape
        if D != cache.head_dim:
            raise TCError(TC_E_ARG, f"head_dim {D} is not the cache's {cache.head_dim}")
        if not (x.is_contiguous() and y.is_contiguous()):
            for i, t in enumerate((x, y)):
                st = t.stride()
                if not t.is_contiguous() and (i >= strided or T != 0 and (st[2] != 1 or (H != 1 and st[1] != D))):
                    raise TCError(TC_E_ARG, "a row's heads are not contiguous" if i < strided else "out is not contiguous")
        dev = torch.cuda.current_device()
        if not x.get_device() == y.get_device() == cache.device == batch.device == dev:
            raise TCError(TC_E_ARG, "tensors are not on the current device")
        return T, self._stream(dev)

    @staticmethod
    def _row_stride(t):
        return _u32(t.stride(0), "row stride") if t.shape[0] > 1 else t.shape[1] * t.shape[2]

    def kv_write(self, cache, batch, k, v):
        """Keys and values [n_tokens][kv_heads][head_dim] (rows may be strided)
        into their slots of the cache."""
        if k.dim() != 3 or k.shape[1] != cache.kv_heads:
            raise TCError(TC_E_ARG, "k is not [n_tokens][kv_heads][head_dim]")
        T, stream = self._kv_call(cache, batch, k, v, 2)
        self._check(self.lib.tc_kv_write(cache.ref, batch.of(T), _elem_type(k.dtype), k.data_ptr(), v.data_ptr(),
                                         self._row_stride(k), self._row_stride(v), stream))

    def kv_read(self, cache, batch, n_tokens, dtype, out=None):
        """The batch's n_tokens rows out of the cache: (k, v)."""
        import torch
        if out is None:
            k = torch.empty((n_tokens, cache.kv_heads, cache.head_dim), dtype=dtype, device=cache.k.device)
            v = torch.empty_like(k)
        else:
            k, v = out
            if k.dim() != 3 or k.shape[:2] != (n_tokens, cache.kv_heads) or k.dtype != dtype:
                raise TCError(TC_E_ARG, "outputs are [n_tokens][kv_heads][head_dim] of dtype")
        T, stream = self._kv_call(cache, batch, k, v, 0)
        self._check(self.lib.tc_kv_read(cache.ref, batch.of(T), _elem_type(dtype), k.data_ptr(), v.data_ptr(), stream))
        return k, v

    def attn(self, cache, batch, q, scale, window=0, out=None):
        """Causal attention of q [n_tokens][heads][head_dim] (rows may be strided)
        over the cache."""
        import torch
        _u32(window, "window")
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        T, stream = self._kv_call(cache, batch, q, out, 1)
        self._check(self.lib.tc_attn(cache.ref, batch.of(T), _elem_type(q.dtype), q.data_ptr(), self._row_stride(q),
                                     out.data_ptr(), q.shape[1], scale, window, stream))
        return out

    def attn_reserve(self, heads, n_tokens):
        self._check(self.lib.tc_attn_reserve(_u32(heads, "heads"), _u32(n_tokens, "n_tokens")))

    def spec_verify(self, logits, tokens, start, temperature, accept_u, sample_u, draft_probs=None):
        """How many of each sequence's drafted tokens hold against the target's
        logits [n_tokens][vocab], and the token after them: (n_accepted, next_token)."""
        import torch
        T, V = logits.shape
        S = temperature.numel()
        dev = torch.cuda.current_device()
        for t in (logits, temperature, accept_u, sample_u, draft_probs):
            if t is not None and (t.dtype != torch.float32 or not t.is_contiguous() or t.get_device() != dev):
                raise TCError(TC_E_ARG, "logits, probabilities and random numbers are contiguous fp32 on the current device")
        for t in (tokens, start):
            if t.dtype != torch.int32 or not t.is_contiguous() or t.get_device() != dev:
                raise TCError(TC_E_ARG, "tokens and start are contiguous int32 on the current device")
        if not (start.numel() == S + 1 and tokens.numel() == accept_u.numel() == T and sample_u.numel() == S and
                (draft_probs is None or draft_probs.shape == logits.shape)):
            raise TCError(TC_E_ARG, "sizes do not agree")
        n = torch.empty(S, dtype=torch.int32, device=logits.device)
        tok = torch.empty_like(n)
        self._check(self.lib.tc_spec_verify(logits.data_ptr(), None if draft_probs is None else draft_probs.data_ptr(), V, S, T,
                                            start.data_ptr(), tokens.data_ptr(), temperature.data_ptr(), accept_u.data_ptr(),
                                            sample_u.data_ptr(), n.data_ptr(), tok.data_ptr(), self._stream(dev)))
        return n, tok

    # -- the rest of a step: geometry, norms, rotary positions, rules on logits ----------
    def kv_plan(self, plan):
        """One step's rows, positions, slots and pages (tc_kv_plan): plan, filled."""
        dev = self._current_device()
        if plan.device != dev:
            raise TCError(TC_E_ARG, "the plan is not on the current device")
        self._check(self.lib.tc_kv_plan(plan.ref, self._stream(dev)))
        return plan

    # (as above, a small call's host time is its whole time: its struct is packed, not built field by field, and
    # outputs are made like a tensor that is there)
    @staticmethod
    def _stride_of(t, T, width):
        """Elements between the rows of t [T][...], each of `width` values next to each other."""
        st, at = t.stride(), 1
        for n, s in zip(t.shape[:0:-1], st[:0:-1]):
            if n != 1 and s != at and T != 0:
                raise TCError(TC_E_ARG, "a row's values are not next to each other")
            at *= n
        return _u32(st[0], "row stride") if T > 1 else width

    def _norm_rows(self, h, y, h_out, x, pre, post, gate, sigmoid, scale, act_type, act):
        shape, dev, types = h.shape, self._current_device(), _ELEM_TYPES
        if len(shape) != 2:
            raise TCError(TC_E_ARG, "h is [rows][cols]")
        T, D = shape
        py = po = px = ys = os_ = xs = ty = tx = 0
        th, good = h.dtype, h.get_device() == dev
        hs = D if h.is_contiguous() else self._stride_of(h, T, D)
        if y is not None:
            py, ty, ys = y.data_ptr(), types.get(y.dtype, -1), D if y.is_contiguous() else self._stride_of(y, T, D)
            good = good and y.shape == shape and y.get_device() == dev
        if h_out is not None:
            po, os_ = h_out.data_ptr(), D if h_out.is_contiguous() else self._stride_of(h_out, T, D)
            good = good and h_out.shape == shape and h_out.dtype == th and h_out.get_device() == dev
        if x is not None:
            px, tx, xs = x.data_ptr(), types.get(x.dtype, -1), D if x.is_contiguous() else self._stride_of(x, T, D)
            good = good and x.shape == shape and x.get_device() == dev
        if not good:
            raise TCError(TC_E_ARG, "rows are [rows][cols] on the current device, h_out of h's type")
        ppre = ppost = pg = kind = tg = 0
        if pre is not None:
            ppre = pre.of(D, dev)
        if post is not None:
            ppost = post.of(D, dev)
        if gate is not None:
            if gate.shape == shape:
                kind = 3
            elif gate.shape == (T, 1):
                kind = 2
            elif gate.shape == (D,):
                kind = 1
            else:
                raise TCError(TC_E_ARG, "a gate is [cols], [rows][1] or [rows][cols]")
            if not gate.is_contiguous() or gate.get_device() != dev:
                raise TCError(TC_E_ARG, "a gate is contiguous, on the current device")
            pg, tg = gate.data_ptr(), types.get(gate.dtype, -1)
        if act is not None and (not act.is_contiguous() or act.get_device() != dev or
                                act.numel() * act.element_size() < self.lib.tc_act_bytes(act_type, T, D)):
            raise TCError(TC_E_ARG, "act is too small, not contiguous or not on the current device")
        c = _PACK_NORM_ROWS(T, D, h.data_ptr(), py, po, px, types.get(th, -1), ty, tx, hs, ys, os_, xs, ppost, ppre, pg, kind, tg,
                            1 if sigmoid else 0, scale, act_type, 0 if act is None else act.data_ptr())
        rc = self.lib.tc_norm_add(c, self._stream(dev))
        if rc:
            self._check(rc)

    def norm(self, h, pre, out_dtype=None, out=None):
        """pre(h): the norm of rows [rows][cols] (which may be strided), of out_dtype (h's)."""
        torch = self._torch
        if out is None:
            out = torch.empty_like(h, dtype=out_dtype, memory_format=torch.contiguous_format)
        self._norm_rows(h, None, None, out, pre, None, None, False, 1.0, 0, None)
        return out

    def norm_add(self, h, y, pre=None, post=None, gate=None, sigmoid=False, scale=1.0, out_dtype=None, h_out=None, out=None,
                 act_type=0, act=None):
        """h + scale * gate * post(y) into h_out (h itself may be given), and pre of that, of
        out_dtype (h's) into out: (h_out, out); without `pre` out is None, without y the first is h. gate [cols],
        [rows][1] or [rows][cols]. act: a buffer of
        tc_act_bytes for the activations quantized for weights of act_type, as act_quantize."""
        torch = self._torch
        if y is None:  # (the call writes no h_out then)
            if h_out is not None and h_out is not h:
                raise TCError(TC_E_ARG, "h_out without the block's output y")
            h_out = h
        elif h_out is None:
            h_out = torch.empty_like(h, memory_format=torch.contiguous_format)
        if out is None and pre is not None:
            out = torch.empty_like(h, dtype=out_dtype, memory_format=torch.contiguous_format)
        self._norm_rows(h, y, h_out, out, pre, post, gate, sigmoid, scale, act_type, act)
        return h_out, out

    def rope(self, rope, x, position, out=None):
        """Rows [n_tokens][heads][head_dim] (which may be strided) rotated at position int32
        [n_tokens]; rows below 0 are left as they are in out (which may be x)."""
        import torch
        if x.dim() != 3:
            raise TCError(TC_E_ARG, "rows are [n_tokens][heads][head_dim]")
        if out is None:
            out = x.clone(memory_format=torch.contiguous_format) if x.shape[0] else torch.empty_like(x)
        T, H, D = x.shape
        dev = torch.cuda.current_device()
        for t in (x, out):
            if t.shape != x.shape or t.dtype != x.dtype or t.get_device() != dev or \
                    (T != 0 and (t.stride(2) != 1 or (H != 1 and t.stride(1) != D))):
                raise TCError(TC_E_ARG, "rows are of one shape and type, a row's heads contiguous, on the current device")
        if position.dtype != torch.int32 or position.shape != (T,) or not position.is_contiguous() or \
                position.get_device() != dev or rope.device != dev:
            raise TCError(TC_E_ARG, "positions are contiguous int32 [n_tokens], they and the rope on the current device")
        self._check(self.lib.tc_rope_apply(rope.ref, _elem_type(x.dtype), x.data_ptr(), self._row_stride(x), out.data_ptr(),
                                           self._row_stride(out), position.data_ptr(), T, H, D, self._stream(dev)))
        return out

    def rope_kv_write(self, cache, batch, rope, q, k, v, q_norm=None, k_norm=None, eps=1e-6, out=None):
        """Queries [n_tokens][heads][head_dim] rotated into out (new, contiguous, or q itself), keys rotated
        and values as they are into their slots of the cache (tc_rope_kv_write). q_norm, k_norm:
        fp32 weights [head_dim] of an RMS norm of the heads before. q may be None."""
        shape, kv, D, dev, dtype = k.shape, cache.kv_heads, cache.head_dim, self._current_device(), k.dtype
        if len(shape) != 3 or shape[1] != kv or shape[2] != D or v.shape != shape or v.dtype != dtype:
            raise TCError(TC_E_ARG, "k and v are not [n_tokens][kv_heads][head_dim] of the cache, of one type")
        T, width, heads, pq, qs, po = shape[0], kv * D, 0, None, 0, None
        ks = width if k.is_contiguous() else self._stride_of(k, T, width)
        vs = width if v.is_contiguous() else self._stride_of(v, T, width)
        good = k.get_device() == v.get_device() == cache.device == batch.device == rope.device == dev
        if q is not None:
            shape = q.shape
            if len(shape) != 3 or shape[0] != T or shape[2] != D or q.dtype != dtype:
                raise TCError(TC_E_ARG, "q is not [n_tokens][heads][head_dim] of k's type")
            if out is None:
                out = self._torch.empty_like(q, memory_format=self._torch.contiguous_format)
            elif out is not q and (out.shape != shape or out.dtype != dtype or out.get_device() != dev or
                                   not (out.stride() == q.stride() if out.data_ptr() == q.data_ptr() else out.is_contiguous())):
                raise TCError(TC_E_ARG, "out is neither q nor like q, contiguous, on the current device")
            heads = shape[1]
            good = good and q.get_device() == dev
            pq, po, qs = q.data_ptr(), out.data_ptr(), heads * D if q.is_contiguous() else self._stride_of(q, T, heads * D)
        elif out is not None:
            raise TCError(TC_E_ARG, "out without q")
        if not good:
            raise TCError(TC_E_ARG, "rows, cache, batch or rope are not on the current device")
        pqn = pkn = None
        if q_norm is not None:
            pqn = self._head_norm(q_norm, D, dev)
        if k_norm is not None:
            pkn = self._head_norm(k_norm, D, dev)
        rc = self.lib.tc_rope_kv_write(cache.ref, batch.of(T), rope.ref, _ELEM_TYPES.get(dtype, -1), pq, qs, po, heads, k.data_ptr(), ks,
                                       v.data_ptr(), vs, pqn, pkn, eps, self._stream(dev))
        if rc:
            self._check(rc)
        return out

    def _head_norm(self, w, D, dev):
        if w.dtype != self._torch.float32 or w.dim() != 1 or w.numel() != D or not w.is_contiguous() or w.get_device() != dev:
            raise TCError(TC_E_ARG, "norms of heads are fp32 [head_dim], contiguous, on the current device")
        return w.data_ptr()

    def logits_adjust(self, rules, logits, start, tokens=None, out=None):
        """Rules on logits [n_tokens][vocab] (rows may be strided) of the sequences' rows start
        int32 [n_seq + 1]: fp32 [n_tokens][vocab] in out (which may be logits). tokens int32
        [n_tokens]: the step's tokens, counted behind the history up to each row's own."""
        shape, dev = logits.shape, self._current_device()
        if out is None:
            out = self._torch.empty_like(logits, dtype=self._torch.float32, memory_format=self._torch.contiguous_format)
        if len(shape) != 2 or out.shape != shape or not logits.get_device() == out.get_device() == dev:
            raise TCError(TC_E_ARG, "logits and out are [n_tokens][vocab] on the current device")
        T, V = shape
        S = start.numel() - 1
        ls = V if logits.is_contiguous() else self._stride_of(logits, T, V)
        os_ = V if out.is_contiguous() else self._stride_of(out, T, V)
        i32, pt = self._torch.int32, None
        good = start.dtype == i32 and start.is_contiguous() and start.get_device() == dev
        if tokens is not None:
            pt = tokens.data_ptr()
            good = good and tokens.dtype == i32 and tokens.numel() == T and tokens.is_contiguous() and tokens.get_device() == dev
        if not good:
            raise TCError(TC_E_ARG, "start and tokens [n_tokens] are contiguous int32 on the current device")
        if out.dtype != self._torch.float32 or S < 0 or (rules.device is not None and rules.device != dev) or \
                (rules.n_seq is not None and rules.n_seq != S) or (rules.rows is not None and rules.rows < T) or \
                (rules.words is not None and rules.words * 32 < V):
            raise TCError(TC_E_ARG, "out is not fp32, or sizes or devices do not agree")
        rc = self.lib.tc_logits_adjust(rules.ref, _ELEM_TYPES.get(logits.dtype, -1), logits.data_ptr(), ls, V, S, T, start.data_ptr(), pt,
                                       out.data_ptr(), os_, self._stream(dev))
        if rc:
            self._check(rc)
        return out


class TensorRecord:
    """One GGUF tensor record (the reference's TensorInfo, IModelLoader.hpp:145:
    name, offset into the data section, shape in file order, GGML type), plus
    its byte size."""

    __slots__ = ("index", "name", "type", "shape", "offset", "bytes")

    def __init__(self, index, name, type_, shape, offset, nbytes):
        self.index, self.name, self.type, self.shape = index, name, type_, shape
        self.offset, self.bytes = offset, nbytes

    def __repr__(self):
        return f"TensorRecord({self.name!r}, type={self.type}, shape={self.shape}, bytes={self.bytes})"


class GGUFLoader:
    """GGUF v3 reader over the C-ABI (tc_gguf_*), shaped like the reference's
    tinycoder::GGUFLoader (include/GGUFLoader.hpp:48): load / loadMetadata,
    getTensor (host bytes, a read-only numpy view of the mapping),
    getTensorInfo, tensorRecords, and upload() to put a tensor's raw blocks in
    device memory for the mat-vec / GEMM entry points. load() returns False on
    failure like the reference; the reason is in last_error."""

    def __init__(self, lib=None):
        self.lib = lib if lib is not None else load_library()
        self.h = None
        self.last_error = ""

    def _open(self, path, fn):
        self.close()
        h = fn(os.fsencode(path))
        if not h:
            self.last_error = self.lib.tc_last_error().decode()
            return False
        self.h = h
        return True

    def load(self, path):
        return self._open(path, self.lib.tc_gguf_open)

    def loadMetadata(self, path):  # noqa: N802 (the reference's name)
        return self._open(path, self.lib.tc_gguf_open_metadata)

    def close(self):
        if self.h:
            self.lib.tc_gguf_close(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @property
    def version(self):
        return self.lib.tc_gguf_version(self.h)

    @property
    def data_offset(self):
        return self.lib.tc_gguf_data_offset(self.h)

    def metadata(self, key):
        v = self.lib.tc_gguf_meta(self.h, key.encode())
        return None if v is None else v.decode("utf-8", "surrogateescape")

    def _record(self, i):
        name = ctypes.c_char_p()
        t, nd = ctypes.c_uint32(), ctypes.c_uint32()
        dims = (ctypes.c_uint64 * 4)()
        off, nb = ctypes.c_uint64(), ctypes.c_uint64()
        rc = self.lib.tc_gguf_tensor_info(self.h, i, ctypes.byref(name), ctypes.byref(t), ctypes.byref(nd),
                                          dims, ctypes.byref(off), ctypes.byref(nb))
        if rc != TC_OK:
            raise TCError(rc, self.lib.tc_last_error().decode())
        return TensorRecord(i, name.value.decode("utf-8", "surrogateescape"), t.value,
                            tuple(dims[k] for k in range(nd.value)), off.value, nb.value)

    def tensorRecords(self):  # noqa: N802
        return [self._record(i) for i in range(self.lib.tc_gguf_tensor_count(self.h))]

    def getTensorInfo(self, name):  # noqa: N802
        i = self.lib.tc_gguf_find_tensor(self.h, name.encode())
        return None if i < 0 else self._record(i)

    def getTensor(self, name):  # noqa: N802
        import numpy as np
        rec = self.getTensorInfo(name)
        if rec is None:
            return None
        p = self.lib.tc_gguf_tensor_data(self.h, rec.index)
        if not p:
            return None
        buf = (ctypes.c_uint8 * rec.bytes).from_address(p)
        a = np.frombuffer(buf, dtype=np.uint8)
        a.flags.writeable = False
        return a

    def upload(self, name, device="cuda"):
        """Raw block bytes of tensor `name` as a uint8 device tensor."""
        import torch
        rec = self.getTensorInfo(name)
        if rec is None:
            raise KeyError(name)
        out = torch.empty(rec.bytes, dtype=torch.uint8, device=device)
        rc = self.lib.tc_gguf_upload(self.h, rec.index, _ptr(out), rec.bytes,
                                     ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        if rc != TC_OK:
            raise TCError(rc, self.lib.tc_last_error().decode())
        return out
