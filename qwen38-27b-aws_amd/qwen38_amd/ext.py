"""ctypes binding of libq38.so (include/q38.h). Device tensors are passed as raw pointers on torch's current HIP stream.

There is no fallback: if the library is missing or was built for another architecture, `library()` raises, and every
step object fails with it. Build it with `python -m qwen38_amd.build` (or `__graft_entry__.build()`).
"""

from __future__ import annotations

import ctypes
from pathlib import Path
from typing import NamedTuple

import torch

from .config import FULL, LINEAR, TextConfig

LIB_PATH = Path(__file__).resolve().parent / "libq38.so"
MAX_LAYERS = 128

EXPORTS = (
    "q38_last_error", "q38_create", "q38_destroy", "q38_buffer_size", "q38_bind", "q38_parity", "q38_set_parity",
    "q38_pack_weight", "q38_pack_weight_fp4", "q38_mxfp4_linear", "q38_fp4_linear", "q38_fp4_linear_scratch", "q38_fp8_linear", "q38_fp8_linear_scratch", "q38_fp8_linear_f32", "q38_fp8_linear_mfma", "q38_fp8_linear_noalloc", "q38_mlp_up", "q38_tiles_size", "q38_verify", "q38_decode", "q38_copy_states", "q38_prefill", "q38_mtp_prefill", "q38_mtp_step", "q38_head_groupmax", "q38_head_pick", "q38_embed", "q38_accept", "q38_spec_step", "q38_spec_step_graph", "q38_verify_step", "q38_step_status",
    "q38_kernel_timer", "q38_paged_append", "q38_paged_attention", "q38_paged_attention_scratch",
)


class Q38Config(ctypes.Structure):
    _fields_ = [
        ("hidden_size", ctypes.c_int), ("intermediate_size", ctypes.c_int), ("vocab_size", ctypes.c_int),
        ("num_layers", ctypes.c_int), ("layer_types", ctypes.c_int * MAX_LAYERS),
        ("num_attention_heads", ctypes.c_int), ("num_key_value_heads", ctypes.c_int), ("head_dim", ctypes.c_int),
        ("rotary_dim", ctypes.c_int),
        ("linear_num_key_heads", ctypes.c_int), ("linear_num_value_heads", ctypes.c_int),
        ("linear_key_head_dim", ctypes.c_int), ("linear_value_head_dim", ctypes.c_int),
        ("linear_conv_kernel_dim", ctypes.c_int), ("rms_norm_eps", ctypes.c_float),
        ("batch_size", ctypes.c_int), ("verify_tokens", ctypes.c_int), ("max_seq_len", ctypes.c_int), ("mtp", ctypes.c_int),
        ("saved_states", ctypes.c_int), ("prefill_chunk", ctypes.c_int), ("weight_format", ctypes.c_int),
        ("kv_cache_format", ctypes.c_int), ("projection_mfma", ctypes.c_int),
        ("kv_pages", ctypes.c_int), ("kv_page_size", ctypes.c_int),
    ]


_lib = None


WEIGHT_FORMATS = {"e4m3": 0, "mxfp4": 1}
KV_CACHE_FORMATS = {"bf16": 0, "fp8": 1}
PROJECTION_MFMA = {"bf16": 0, "fp8": 1}


def library() -> ctypes.CDLL:
    """The loaded libq38.so with argument types set. Raises if it is not built."""
    global _lib
    if _lib is not None:
        return _lib
    if not LIB_PATH.exists():
        raise RuntimeError(f"{LIB_PATH} is not built: run `python -m qwen38_amd.build` (the verify path has no fallback)")
    lib = ctypes.CDLL(str(LIB_PATH))
    p, i, sz = ctypes.c_void_p, ctypes.c_int, ctypes.c_size_t
    lib.q38_last_error.restype = ctypes.c_char_p
    lib.q38_last_error.argtypes = []
    lib.q38_create.argtypes = [ctypes.POINTER(Q38Config), ctypes.POINTER(p)]
    lib.q38_destroy.argtypes = [p]
    lib.q38_destroy.restype = None
    lib.q38_buffer_size.argtypes = [p, ctypes.c_char_p, i, ctypes.POINTER(sz)]
    lib.q38_bind.argtypes = [p, ctypes.c_char_p, i, p, sz]
    lib.q38_parity.argtypes = [p, ctypes.POINTER(i)]
    lib.q38_set_parity.argtypes = [p, i]
    lib.q38_pack_weight.argtypes = [p, p, i, i, p, p, p]
    lib.q38_pack_weight_fp4.argtypes = [p, p, i, i, p, p, p]
    lib.q38_fp8_linear.argtypes = [p, i, i, p, p, i, p, p, p]
    lib.q38_mxfp4_linear.argtypes = [p, i, i, p, p, i, p, p, p]
    lib.q38_fp4_linear.argtypes = [p, i, i, p, p, i, p, p, p]
    lib.q38_fp4_linear_scratch.argtypes = [i, i]
    lib.q38_fp8_linear_scratch.argtypes = [i, i]
    lib.q38_fp8_linear_f32.argtypes = [p, i, i, p, p, i, p, p, p]
    lib.q38_fp8_linear_mfma.argtypes = [p, i, i, p, p, i, i, i, p, p, p]
    lib.q38_fp8_linear_noalloc.argtypes = [p, i, i, p, p, i, p, p]
    lib.q38_mlp_up.argtypes = [p, i, i, p, p, i, p, p, p]
    lib.q38_tiles_size.argtypes = [i, i]
    lib.q38_kernel_timer.argtypes = [p, i, ctypes.POINTER(i), ctypes.POINTER(ctypes.c_float)]
    lib.q38_verify.argtypes = [p] * 8 + [p]
    lib.q38_decode.argtypes = [p] * 8
    lib.q38_copy_states.argtypes = [p, p, i, p]
    lib.q38_prefill.argtypes = [p, p, p, p, p, p, p, i, p, p]
    lib.q38_mtp_prefill.argtypes = [p, p, p, p, p, p, p, i, p, p]
    lib.q38_mtp_step.argtypes = [p] * 8 + [p]
    lib.q38_head_groupmax.argtypes = [p, p, i, p, p]
    lib.q38_head_pick.argtypes = [p, p, i, i, p, p]
    lib.q38_embed.argtypes = [p, p, i, p, p]
    lib.q38_accept.argtypes = [p, p, p, p, p, p, p]
    lib.q38_spec_step.argtypes = [p] * 10
    lib.q38_spec_step_graph.argtypes = [p] * 10
    lib.q38_verify_step.argtypes = [p] * 10
    lib.q38_step_status.argtypes = [p, ctypes.POINTER(i), i, p]
    lib.q38_paged_append.argtypes = [p, p, p, p]
    lib.q38_paged_attention.argtypes = [p, p, p, p, sz, p]
    lib.q38_paged_attention_scratch.argtypes = [p, p, i]
    sizes = ("q38_fp8_linear_scratch", "q38_fp4_linear_scratch", "q38_tiles_size", "q38_paged_attention_scratch")
    for name in EXPORTS:
        if name not in ("q38_last_error", "q38_destroy"):
            getattr(lib, name).restype = ctypes.c_size_t if name in sizes else ctypes.c_int
    _lib = lib
    return lib


def check(rc: int) -> None:
    if rc:
        raise RuntimeError("libq38: " + library().q38_last_error().decode())


def ptr(t: torch.Tensor | None) -> int | None:
    if t is None:
        return None
    if not t.is_cuda:
        raise ValueError("libq38 takes device tensors")
    if not t.is_contiguous():
        raise ValueError("libq38 takes contiguous tensors")
    return t.data_ptr()


def stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def make_config(cfg: TextConfig, batch: int, tokens: int, max_seq_len: int, mtp: bool, saved_states: bool = False,
                prefill_chunk: int = 0, weight_format: str = "e4m3", kv_cache_format: str = "bf16",
                projection_mfma: str = "bf16", kv_pages: int = 0, kv_page_size: int = 64) -> Q38Config:
    c = Q38Config()
    c.hidden_size, c.intermediate_size, c.vocab_size = cfg.hidden_size, cfg.intermediate_size, cfg.vocab_size
    if cfg.num_hidden_layers > MAX_LAYERS:
        raise ValueError(f"at most {MAX_LAYERS} layers")
    c.num_layers = cfg.num_hidden_layers
    for i, kind in enumerate(cfg.layer_types):
        c.layer_types[i] = {LINEAR: 0, FULL: 1}[kind]
    c.num_attention_heads, c.num_key_value_heads, c.head_dim = cfg.num_attention_heads, cfg.num_key_value_heads, cfg.head_dim
    c.rotary_dim = cfg.rotary_dim
    c.linear_num_key_heads, c.linear_num_value_heads = cfg.linear_num_key_heads, cfg.linear_num_value_heads
    c.linear_key_head_dim, c.linear_value_head_dim = cfg.linear_key_head_dim, cfg.linear_value_head_dim
    c.linear_conv_kernel_dim = cfg.linear_conv_kernel_dim
    c.rms_norm_eps = cfg.rms_norm_eps
    c.batch_size, c.verify_tokens, c.max_seq_len, c.mtp = batch, tokens, max_seq_len, int(mtp)
    c.saved_states = int(saved_states)
    c.prefill_chunk = prefill_chunk
    c.weight_format = WEIGHT_FORMATS[weight_format]
    c.kv_cache_format = KV_CACHE_FORMATS[kv_cache_format]
    c.projection_mfma = PROJECTION_MFMA[projection_mfma]
    c.kv_pages, c.kv_page_size = kv_pages, kv_page_size
    return c


class Handle:
    """One q38_handle: shapes fixed at creation, every buffer bound by the owner."""

    def __init__(self, cfg: TextConfig, batch: int, tokens: int, max_seq_len: int, mtp: bool, saved_states: bool = False,
                 prefill_chunk: int = 0, weight_format: str = "e4m3", kv_cache_format: str = "bf16", projection_mfma: str = "bf16",
                 kv_pages: int = 0, kv_page_size: int = 64):
        self.lib = library()
        self.c = make_config(cfg, batch, tokens, max_seq_len, mtp, saved_states, prefill_chunk, weight_format, kv_cache_format,
                             projection_mfma, kv_pages, kv_page_size)
        h = ctypes.c_void_p()
        check(self.lib.q38_create(ctypes.byref(self.c), ctypes.byref(h)))
        self.h = h

    def __del__(self):
        if getattr(self, "h", None) and self.h.value:
            self.lib.q38_destroy(self.h)
            self.h = None

    def buffer_size(self, name: str, layer: int) -> int:
        n = ctypes.c_size_t()
        check(self.lib.q38_buffer_size(self.h, name.encode(), layer, ctypes.byref(n)))
        return n.value

    def bind(self, name: str, layer: int, t: torch.Tensor) -> None:
        check(self.lib.q38_bind(self.h, name.encode(), layer, ptr(t), t.numel() * t.element_size()))

    @property
    def parity(self) -> int:
        p = ctypes.c_int()
        check(self.lib.q38_parity(self.h, ctypes.byref(p)))
        return p.value

    @parity.setter
    def parity(self, value: int) -> None:
        check(self.lib.q38_set_parity(self.h, value))

    def verify(self, embeds, cos, sin, position, active, accepted, out) -> None:
        check(self.lib.q38_verify(self.h, *map(ptr, (embeds, cos, sin, position, active, accepted, out)), stream()))

    def decode(self, embeds, cos, sin, position, active, out) -> None:
        check(self.lib.q38_decode(self.h, *map(ptr, (embeds, cos, sin, position, active, out)), stream()))

    def prefill(self, embeds, cos, sin, slot, start, n_valid, tokens: int, out) -> None:
        check(self.lib.q38_prefill(self.h, *map(ptr, (embeds, cos, sin, slot, start, n_valid)), tokens, ptr(out), stream()))

    def mtp_prefill(self, hidden, embeds, cos, sin, slot, start, tokens: int, out) -> None:
        check(self.lib.q38_mtp_prefill(self.h, *map(ptr, (hidden, embeds, cos, sin, slot, start)), tokens, ptr(out), stream()))

    def copy_states(self, slot, to_saved: bool) -> None:
        check(self.lib.q38_copy_states(self.h, ptr(slot), int(to_saved), stream()))

    def mtp_step(self, hidden, embeds, cos, sin, position, active, out) -> None:
        check(self.lib.q38_mtp_step(self.h, *map(ptr, (hidden, embeds, cos, sin, position, active, out)), stream()))

    def head_groupmax(self, hidden, rows: int, maxima) -> None:
        check(self.lib.q38_head_groupmax(self.h, ptr(hidden), rows, ptr(maxima), stream()))

    def head_pick(self, hidden, rows: int, groups: int, ids) -> None:
        check(self.lib.q38_head_pick(self.h, ptr(hidden), rows, groups, ptr(ids), stream()))

    def embed(self, ids, n: int, out) -> None:
        check(self.lib.q38_embed(self.h, ptr(ids), n, ptr(out), stream()))

    def accept(self, picks, drafts, active, match, accepted) -> None:
        check(self.lib.q38_accept(self.h, *map(ptr, (picks, drafts, active, match, accepted)), stream()))

    def spec_step(self, position, index, match, accepted, active, hidden, picks, drafts, graph: bool = False) -> None:
        """One speculative step on the device (`q38_spec_step`), or its captured HIP graph (`q38_spec_step_graph`)."""
        fn = self.lib.q38_spec_step_graph if graph else self.lib.q38_spec_step
        check(fn(self.h, *map(ptr, (position, index, match, accepted, active, hidden, picks, drafts)), stream()))

    def verify_step(self, position, index, match, accepted, active, hidden, picks, drafts) -> None:
        """The verify half of the speculative step for host-made drafts (`q38_verify_step`): the prompt-lookup
        branch of the reference's `Scheduler._verify_step` (scheduler.py:269-301)."""
        check(self.lib.q38_verify_step(self.h, *map(ptr, (position, index, match, accepted, active, hidden, picks, drafts)),
                                       stream()))

    def step_status(self, clear: bool = True) -> int:
        """The device's step status word (`q38_step_status`: STATUS_NONFINITE, STATUS_POSITION), then reset."""
        v = ctypes.c_int(0)
        check(self.lib.q38_step_status(self.h, ctypes.byref(v), int(clear), stream()))
        return v.value

    def raise_step_errors(self) -> None:
        """The reference's host-side errors for what the last steps recorded on the device: FloatingPointError for a
        row with no finite logit (generate.py:206-207), ValueError for tokens past the last usable position
        (generate.py:78-79)."""
        status = self.step_status()
        if status & STATUS_NONFINITE:
            raise FloatingPointError("a row's logits are not finite, so the step produced NaN or infinity")
        if status & STATUS_POSITION:
            raise ValueError("a row's tokens pass max_seq_len")

    def kernel_timer(self, on: bool) -> tuple[int, float]:
        """Start (on) or stop bracketing the gate/up GEMM launches with HIP events; stopping returns (launches, total
        milliseconds)."""
        n, ms = ctypes.c_int(0), ctypes.c_float(0.0)
        check(self.lib.q38_kernel_timer(self.h, int(on), ctypes.byref(n), ctypes.byref(ms)))
        return n.value, ms.value


def pack_weight(coded: torch.Tensor, scales: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(e4m3 bytes [N, K], E8M0 bytes [N, K/32]) on the GPU -> (tiles, tile scales) in the GEMM layout."""
    n, k = coded.shape
    tiles = torch.empty(n * k, dtype=torch.uint8, device=coded.device)
    tile_scales = torch.empty(n * k // 32, dtype=torch.uint8, device=coded.device)
    check(library().q38_pack_weight(ptr(coded.contiguous()), ptr(scales.contiguous()), n, k, ptr(tiles), ptr(tile_scales), stream()))
    return tiles, tile_scales


def pack_weight_fp4(packed: torch.Tensor, scales: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The checkpoint's MXFP4 (packed bytes [N, K/2], E8M0 bytes [N, K/32]) on the GPU -> (tiles, tile scales)."""
    n, half = packed.shape
    k = 2 * half
    tiles = torch.empty(n * half, dtype=torch.uint8, device=packed.device)
    tile_scales = torch.empty(n * k // 32, dtype=torch.uint8, device=packed.device)
    check(library().q38_pack_weight_fp4(ptr(packed.contiguous()), ptr(scales.contiguous()), n, k, ptr(tiles), ptr(tile_scales),
                                        stream()))
    return tiles, tile_scales


def linear_scratch(rows: int, k: int, device="cuda") -> torch.Tensor:
    """Zero-filled scratch for the standalone projections (input tiles, then the GEMM's counters and partials)."""
    return torch.zeros(library().q38_fp8_linear_scratch(rows, k), dtype=torch.uint8, device=device)


def fp8_linear(x: torch.Tensor, tiles: torch.Tensor, scales: torch.Tensor, n: int, scratch=None) -> torch.Tensor:
    """`FP8Linear.forward` on the GPU: bf16 x [rows, k] -> bf16 [rows, n] through a packed FP8 weight."""
    rows, k = x.shape
    scratch = linear_scratch(rows, k, x.device) if scratch is None else scratch
    out = torch.empty(rows, n, dtype=torch.bfloat16, device=x.device)
    check(library().q38_fp8_linear(ptr(x.contiguous()), rows, k, ptr(tiles), ptr(scales), n, ptr(scratch), ptr(out), stream()))
    return out


def fp8_linear_noalloc(x: torch.Tensor, tiles: torch.Tensor, scales: torch.Tensor, n: int, out=None) -> torch.Tensor:
    """`fp8_linear` with the library's static scratch (no device allocation by the library): 1 to 64 rows."""
    rows, k = x.shape
    out = torch.empty(rows, n, dtype=torch.bfloat16, device=x.device) if out is None else out
    check(library().q38_fp8_linear_noalloc(ptr(x.contiguous()), rows, k, ptr(tiles), ptr(scales), n, ptr(out), stream()))
    return out


GEMM_RECOMPUTE = 4  # Q38_GEMM_RECOMPUTE
STATUS_NONFINITE, STATUS_POSITION = 1, 2  # Q38_STATUS_*


def fp8_linear_mfma(x: torch.Tensor, tiles: torch.Tensor, scales: torch.Tensor, n: int, mfma: str, f32_out: bool = False,
                    scratch=None, recompute: bool = False) -> torch.Tensor:
    """The FP8 projection with its products on the named MFMA ("fp8" or "bf16"), bf16 or float32 output; with
    ``recompute`` every tile split between workgroups is finished by recomputing its partials (the GEMM's path for
    contributors on different XCDs)."""
    rows, k = x.shape
    scratch = linear_scratch(rows, k, x.device) if scratch is None else scratch
    out = torch.empty(rows, n, dtype=torch.float32 if f32_out else torch.bfloat16, device=x.device)
    flags = PROJECTION_MFMA[mfma] | (GEMM_RECOMPUTE if recompute else 0)
    check(library().q38_fp8_linear_mfma(ptr(x.contiguous()), rows, k, ptr(tiles), ptr(scales), n, flags,
                                        int(f32_out), ptr(scratch), ptr(out), stream()))
    return out


def mxfp4_linear(x: torch.Tensor, tiles: torch.Tensor, scales: torch.Tensor, n: int, scratch=None) -> torch.Tensor:
    """The projection through a packed MXFP4 weight (`pack_weight_fp4`): bf16 x [rows, k] -> bf16 [rows, n]."""
    rows, k = x.shape
    scratch = linear_scratch(rows, k, x.device) if scratch is None else scratch
    out = torch.empty(rows, n, dtype=torch.bfloat16, device=x.device)
    check(library().q38_mxfp4_linear(ptr(x.contiguous()), rows, k, ptr(tiles), ptr(scales), n, ptr(scratch), ptr(out), stream()))
    return out


def fp4_linear(x: torch.Tensor, tiles: torch.Tensor, scales: torch.Tensor, n: int, scratch=None) -> torch.Tensor:
    """`FP4Linear.forward` on the GPU (the weight_format "fp4" numerics): bf16 x [rows, k] -> bf16 [rows, n] through a
    packed MXFP4 weight (`pack_weight_fp4`), the even and odd inputs summed apart and their bf16 results added."""
    rows, k = x.shape
    if scratch is None:
        scratch = torch.zeros(library().q38_fp4_linear_scratch(rows, k), dtype=torch.uint8, device=x.device)
    out = torch.empty(rows, n, dtype=torch.bfloat16, device=x.device)
    check(library().q38_fp4_linear(ptr(x.contiguous()), rows, k, ptr(tiles), ptr(scales), n, ptr(scratch), ptr(out), stream()))
    return out


def fp8_linear_f32(x: torch.Tensor, tiles: torch.Tensor, scales: torch.Tensor, n: int, scratch=None) -> torch.Tensor:
    """The FP8 projection with float32 output (no bf16 rounding): rows in {32, 64, 128} or a multiple of 256."""
    rows, k = x.shape
    scratch = linear_scratch(rows, k, x.device) if scratch is None else scratch
    out = torch.empty(rows, n, dtype=torch.float32, device=x.device)
    check(library().q38_fp8_linear_f32(ptr(x.contiguous()), rows, k, ptr(tiles), ptr(scales), n, ptr(scratch), ptr(out), stream()))
    return out


def mlp_up(x: torch.Tensor | None, rows: int, k: int, tiles: torch.Tensor, scales: torch.Tensor, inter: int, scratch=None,
           out=None) -> torch.Tensor:
    """The fused gate/up projection with SwiGLU (`mlp_up`): bf16 x [rows, k] -> the down projection's e5m2 input tiles.
    With x None the scratch already holds the input tiles of an earlier call."""
    lib = library()
    if scratch is None:
        scratch = linear_scratch(rows, k)
    if out is None:
        out = torch.empty(lib.q38_tiles_size(rows, inter), dtype=torch.uint8, device=scratch.device)
    xp = None if x is None else ptr(x.contiguous())
    check(lib.q38_mlp_up(xp, rows, k, ptr(tiles), ptr(scales), inter, ptr(scratch), ptr(out), stream()))
    return out


# ------------------------------------------------------------------------------------------------ the paged 8-bit cache


class PagedCache(NamedTuple):
    """One layer's keys and values in pages of 8-bit values (`q38_paged_cache`): k uint8 (e4m3) [pages, kv_heads, page, hd], v uint8
    (e4m3) [pages, kv_heads, page / 16, hd, 16], k_scale, v_scale uint8 (E8M0) [pages, kv_heads]. `paged_cache` makes one."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


def paged_cache(pages: int, kv_heads: int, head_dim: int, page_size: int = 64, device="cuda") -> PagedCache:
    """An empty cache: zeros, every page's scale 1."""
    zeros = lambda *shape: torch.zeros(*shape, dtype=torch.uint8, device=device)  # noqa: E731
    return PagedCache(zeros(pages, kv_heads, page_size, head_dim), zeros(pages, kv_heads, page_size // 16, head_dim, 16),
                      zeros(pages, kv_heads) + 127, zeros(pages, kv_heads) + 127)


def paged_values(cache: PagedCache) -> tuple[torch.Tensor, torch.Tensor]:
    """What a cache holds as float32: keys and values [pages, kv_heads, page, hd]."""
    times = lambda b: torch.ldexp(torch.ones((), device=b.device), b.int() - 127)[:, :, None, None]  # noqa: E731
    e4m3 = lambda x: x.view(torch.float8_e4m3fn).float()  # noqa: E731
    return e4m3(cache.k) * times(cache.k_scale), e4m3(cache.v).transpose(-1, -2).flatten(2, 3) * times(cache.v_scale)


class _CacheArgs(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("k", "v", "k_scale", "v_scale")] + [
        (n, ctypes.c_int) for n in ("pages", "kv_heads", "head_dim", "page_size")]


class _RowArgs(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("position", "pages", "q_start")] + [
        (n, ctypes.c_int) for n in ("rows", "max_pages", "tokens", "max_tokens")]


class _TokenArgs(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("k", "v", "q", "q_out")]
                + [(n, ctypes.c_longlong) for n in ("k_token", "k_head", "v_token", "v_head", "q_token", "q_head")]
                + [("q_heads", ctypes.c_int), ("rotary_dim", ctypes.c_int)]
                + [(n, ctypes.c_void_p) for n in ("cos", "sin", "q_norm", "k_norm")] + [("eps", ctypes.c_float)])


class _QueryArgs(ctypes.Structure):
    _fields_ = [("q", ctypes.c_void_p), ("out", ctypes.c_void_p), ("q_heads", ctypes.c_int), ("scale", ctypes.c_float),
                ("cap", ctypes.c_float), ("window", ctypes.c_int), ("slopes", ctypes.c_void_p), ("prefix", ctypes.c_void_p)]


def _want(name: str, t: torch.Tensor, dtype: torch.dtype, shape: tuple, device: int) -> int:
    """The pointer of a contiguous tensor of this type and shape on this device (its index); ValueError if it is another."""
    if t.dtype is dtype and t.shape == shape and t.get_device() == device and t.is_contiguous():
        return t.data_ptr()
    raise ValueError(f"{name} must be contiguous {dtype} {list(shape)} on device {device}, got {t.dtype} {list(t.shape)} on {t.device}")


def _heads_of(name: str, t: torch.Tensor, tokens: int, head_dim: int, device: int) -> tuple[int, int, int]:
    """Pointer and token and head strides of bf16 [tokens, heads, head_dim] whose last dim is contiguous."""
    if t.dtype is not torch.bfloat16 or t.dim() != 3 or t.shape[0] != tokens or t.shape[2] != head_dim or t.get_device() != device:
        raise ValueError(f"{name} must be torch.bfloat16 [{tokens}, heads, {head_dim}] on device {device}, got {t.dtype} {list(t.shape)} on {t.device}")
    token, head, one = t.stride()
    if one != 1:
        raise ValueError(f"{name}'s last dim must be contiguous")
    return t.data_ptr(), token, head


def _paged_args(cache: PagedCache, position: torch.Tensor, pages: torch.Tensor, tokens: int, q_start, max_tokens):
    """The cache and the rows of a call as the library takes them, and the index of their device."""
    k = cache.k
    if not k.is_cuda or k.dim() != 4:
        raise ValueError("the cache must be on a device, its keys [pages, kv_heads, page, head_dim]")
    device, u8, i32 = k.get_device(), torch.uint8, torch.int32
    count, heads, size, hd = k.shape
    c = _CacheArgs(_want("cache.k", k, u8, (count, heads, size, hd), device), _want("cache.v", cache.v, u8, (count, heads, size // 16, hd, 16), device),
                   _want("cache.k_scale", cache.k_scale, u8, (count, heads), device),
                   _want("cache.v_scale", cache.v_scale, u8, (count, heads), device), count, heads, hd, size)
    if pages.dim() != 2:
        raise ValueError(f"pages must be [rows, max_pages], got {list(pages.shape)}")
    rows, width = pages.shape
    if q_start is None:
        if rows < 1 or tokens % rows:
            raise ValueError(f"{tokens} tokens are not the same number in each of {rows} rows: say where they start (q_start)")
        start, max_tokens = None, tokens // rows
    elif max_tokens is None:
        raise ValueError("ragged rows (q_start) need max_tokens, the most tokens of a row")
    else:
        start, max_tokens = _want("q_start", q_start, i32, (rows + 1,), device), min(max_tokens, tokens)
    return c, _RowArgs(_want("position", position, i32, (rows,), device), _want("pages", pages, i32, (rows, width), device), start, rows, width,
                       tokens, max_tokens), device


def _on(device: int, fn, *args) -> None:
    """fn(*args, stream) with the device's current stream (its number as torch's own code asks for it: `stream` takes longer than
    the rest of a small call's checks)."""
    if device != torch._C._cuda_getDevice():
        with torch.cuda.device(device):
            return _on(device, fn, *args)
    check(fn(*args, torch._C._cuda_getCurrentRawStream(device)))


def paged_append(cache: PagedCache, k: torch.Tensor, v: torch.Tensor, position: torch.Tensor, pages: torch.Tensor, *, cos=None, sin=None,
                 q=None, q_start=None, max_tokens: int | None = None, q_norm=None, k_norm=None, eps: float = 1e-6, q_out=None):
    """Append bf16 keys and values [tokens, kv_heads, hd] to the rows' pages (`q38_paged_append`): normed (k_norm) and rotated (cos,
    sin bf16 [tokens, rotary_dim]) on the way, coded to e4m3 with a power of two per page and head. position int32 [rows] is each
    row's first new position (negative: the row is skipped), pages int32 [rows, max_pages] its page table, q_start int32 [rows + 1]
    where its tokens start (None: the same number in each row; else max_tokens is the most that a row has). With queries q
    [tokens, q_heads, hd] they are normed and rotated beside the keys and returned (in q_out, or a new tensor)."""
    tokens, bf = k.shape[0], torch.bfloat16
    c, r, device = _paged_args(cache, position, pages, tokens, q_start, max_tokens)
    hd, rot = c.head_dim, 0
    kp, k_token, k_head = _heads_of("k", k, tokens, hd, device)
    vp, v_token, v_head = _heads_of("v", v, tokens, hd, device)
    if k.shape[1] != c.kv_heads or v.shape[1] != c.kv_heads:
        raise ValueError(f"keys and values of {c.kv_heads} heads, got {k.shape[1]} and {v.shape[1]}")
    if cos is None:
        if sin is not None:
            raise ValueError("cos and sin go together")
        cp = sp = None
    else:
        if sin is None or cos.dim() != 2:
            raise ValueError("cos and sin go together, [tokens, rotary_dim]")
        rot = cos.shape[1]
        cp, sp = _want("cos", cos, bf, (tokens, rot), device), _want("sin", sin, bf, (tokens, rot), device)
    kn = None if k_norm is None else _want("k_norm", k_norm, bf, (hd,), device)
    if q is None:
        if q_norm is not None or q_out is not None:
            raise ValueError("q_norm and q_out need q")
        t = _TokenArgs(kp, vp, None, None, k_token, k_head, v_token, v_head, 0, 0, 0, rot, cp, sp, None, kn, eps)
    else:
        qp, q_token, q_head = _heads_of("q", q, tokens, hd, device)
        heads = q.shape[1]
        if q_out is None:
            q_out = torch.empty(tokens, heads, hd, dtype=bf, device=k.device)
        t = _TokenArgs(kp, vp, qp, _want("q_out", q_out, bf, (tokens, heads, hd), device), k_token, k_head, v_token, v_head, q_token, q_head, heads,
                       rot, cp, sp, None if q_norm is None else _want("q_norm", q_norm, bf, (hd,), device), kn, eps)
    ref = ctypes.byref
    _on(device, library().q38_paged_append, ref(c), ref(r), ref(t))
    return q_out


def paged_attention(cache: PagedCache, q: torch.Tensor, position: torch.Tensor, pages: torch.Tensor, *, q_start=None, max_tokens: int | None = None,
                    scale: float | None = None, cap: float = 0.0, slopes=None, window: int = 0, prefix=None, out=None, scratch=None):
    """Attention of bf16 queries [tokens, q_heads, hd] over their rows' pages, the queries' own positions among them (appended
    before; rows as `paged_append` takes them): `q38_paged_attention`. scale None is hd ** -0.5; cap > 0 caps the scores by
    cap * tanh(score / cap); slopes float32 [q_heads] add slope * (j - i); window > 0 sees the last `window` positions; prefix int32
    [rows]: positions below it are seen by every token. Returns bf16 [tokens, q_heads, hd] (in out, or a new tensor)."""
    if q.dim() != 3:
        raise ValueError(f"q must be [tokens, q_heads, hd], got {list(q.shape)}")
    tokens, heads, hd = q.shape
    c, r, device = _paged_args(cache, position, pages, tokens, q_start, max_tokens)
    bf, shape = torch.bfloat16, (tokens, heads, c.head_dim)
    qp = _want("q", q, bf, shape, device)
    if out is None:
        out = torch.empty(shape, dtype=bf, device=q.device)
    a = _QueryArgs(qp, _want("out", out, bf, shape, device), heads, hd**-0.5 if scale is None else scale, cap, window,
                   None if slopes is None else _want("slopes", slopes, torch.float32, (heads,), device),
                   None if prefix is None else _want("prefix", prefix, torch.int32, (r.rows,), device))
    if not 0 <= window < 2**31:
        raise ValueError(f"window must be 0 (none) to 2**31 - 1, got {window}")
    ref, lib = ctypes.byref, library()
    if scratch is None:
        size = lib.q38_paged_attention_scratch(ref(c), ref(r), heads)
        scratch = torch.empty(size, dtype=torch.uint8, device=q.device)
    else:
        size = scratch.numel() * scratch.element_size()
    _on(device, lib.q38_paged_attention, ref(c), ref(r), ref(a), _want("scratch", scratch, scratch.dtype, scratch.shape, device), size)
    return out
