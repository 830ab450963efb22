"""An 8-bit paged key/value cache and the attention over it.

`KVCache` holds the keys and values of a batch of sequences as float8 e4m3 or
int8 codes, in pages of `page_size` tokens, with one power-of-two scale for each
page and head (include/ttjam_b200.h states the format). Three calls work on one
layer of it, each on `torch.cuda.current_stream()` without a host sync:

* `write(k, v)` quantises the keys and values of new tokens into it;
* `attend(q)` is the causal attention of the new tokens over it;
* `read()` gives the tokens back as dense tensors.

`advance(tokens)` makes room first: it adds the new tokens to `lengths`, and the
calls on all layers then take row i of a sequence's `count` new ones to stand at
position `lengths - count + i`. `UserOptimizedTransformer.forward_cached` does
all of this for a whole model.

There is no CPU path and no autograd: the cache is for running a model, and
CPU tensors raise. The reference has no counterpart; it computes every key and
value anew on each forward (torch_transformer_benchmark.py:93-121).
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import _lib

FORMATS = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
PAGE_SIZES = (16, 32, 64, 128)


def _dtype_code(t: torch.Tensor, what: str) -> int:
    code = _lib.DTYPE_CODES.get(str(t.dtype).split(".")[-1])
    if code is None:
        raise ValueError(f"{what} must be float32, float16 or bfloat16, got {t.dtype}")
    return code


class KVCache:
    """Keys and values of `batch` sequences of up to `max_tokens` tokens, for
    `num_layers` layers of `kv_heads` heads.

    The tensors are public: `k` and `v` are [num_layers, num_pages, kv_heads,
    page_size, head_dim] codes (torch.float8_e4m3fn or torch.int8), `k_scale`
    and `v_scale` [num_layers, num_pages, kv_heads] float32, `block_table`
    [batch, max_tokens / page_size, rounded up] int32 and `lengths` [batch] int32.
    The constructor gives every sequence pages of its own; a program with its
    own page allocator writes into `block_table` and `lengths`, or brings its
    tensors (`from_tensors`). Sequences may share pages that are only read.
    The tensors themselves are fixed for the cache's life (their contents change)."""

    def __init__(self, batch: int, max_tokens: int, kv_heads: int, head_dim: int, *,
                 num_layers: int = 1, page_size: int = 64, fmt: str = "e4m3",
                 device=None) -> None:
        if fmt not in FORMATS:
            raise ValueError(f"fmt must be one of {sorted(FORMATS)}, got {fmt!r}")
        for name, n in (("batch", batch), ("max_tokens", max_tokens), ("kv_heads", kv_heads),
                        ("head_dim", head_dim), ("num_layers", num_layers)):
            if n <= 0:
                raise ValueError(f"{name} must be positive")
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
        device = torch.device("cuda" if device is None else device)
        if device.type != "cuda":
            raise RuntimeError("KVCache runs on CUDA only (no CPU path)")
        columns = -(-max_tokens // page_size)
        pages = batch * columns
        shape = (num_layers, pages, kv_heads, page_size, head_dim)
        codes = [torch.zeros(shape, dtype=torch.uint8, device=device).view(FORMATS[fmt])
                 for _ in range(2)]
        scales = [torch.zeros(shape[:3], dtype=torch.float32, device=device) for _ in range(2)]
        table = torch.arange(pages, dtype=torch.int32, device=device).view(batch, columns)
        with torch.inference_mode(False):  # so that torch counts the writes into it
            lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self._setup(*codes, *scales, table, lengths, max_tokens)
        self._longest, self._seen = 0, lengths._version

    @classmethod
    def from_tensors(cls, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor,
                     v_scale: torch.Tensor, block_table: torch.Tensor,
                     lengths: torch.Tensor) -> "KVCache":
        """A cache over the caller's tensors, of the shapes and types the class
        names (all contiguous, on one device). Scales are powers of two: those
        that `write` made, or a copy of them; others count as NaN in `attend`,
        and in `write` to the middle of their page (`read_device_status`)."""
        self = cls.__new__(cls)
        if block_table.dim() != 2 or k.dim() != 5:
            raise ValueError("k must be [layers, pages, kv_heads, page_size, head_dim] and "
                             "block_table [batch, columns]")
        self._setup(k, v, k_scale, v_scale, block_table, lengths,
                    block_table.shape[1] * k.shape[3])
        return self

    def _setup(self, k, v, k_scale, v_scale, block_table, lengths, max_tokens) -> None:
        fmt = {t: f for f, t in FORMATS.items()}.get(k.dtype)
        if fmt is None:
            raise ValueError(f"codes must be torch.float8_e4m3fn or torch.int8, got {k.dtype}")
        layers, pages, heads, page, hd = k.shape
        batch, columns = block_table.shape
        if page not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page}")
        want = {"v": (v, k.shape, k.dtype), "k_scale": (k_scale, k.shape[:3], torch.float32),
                "v_scale": (v_scale, k.shape[:3], torch.float32),
                "block_table": (block_table, (batch, columns), torch.int32),
                "lengths": (lengths, (batch,), torch.int32)}
        for name, (t, shape, dtype) in {"k": (k, k.shape, k.dtype), **want}.items():
            if t.device.type != "cuda":
                raise RuntimeError("KVCache runs on CUDA only (no CPU path)")
            if (tuple(t.shape) != tuple(shape) or t.dtype != dtype or t.device != k.device
                    or not t.is_contiguous()):
                raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape "
                                 f"{tuple(shape)} on {k.device}, got {t.dtype} of "
                                 f"{tuple(t.shape)} on {t.device}")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.block_table, self.lengths = block_table, lengths
        self.fmt, self.device = fmt, k.device
        self.num_layers, self.num_pages = layers, pages
        self.kv_heads, self.page_size, self.head_dim = heads, page, hd
        self.batch, self.max_tokens = batch, max_tokens
        # An upper bound on lengths, which holds as long as nothing else has written into
        # them: torch's count of the writes is still _seen. None: the bound is not kept.
        self._longest, self._seen = 0, None
        self._status = torch.zeros(2, dtype=torch.int32, device=k.device)
        self._lib = _lib.load()
        self._c_write, self._c_read = self._lib.tt_kv_write, self._lib.tt_kv_read
        self._c_attend = self._lib.tt_kv_attention
        self._index, self._scale = k.device.index, hd ** -0.5
        self._plans = {}
        self._array = (_lib.TTKVCache * layers)()  # one entry a layer
        self._structs = [ctypes.pointer(c) for c in self._array]
        for i, c in enumerate(self._array):
            c.k_codes, c.v_codes = k[i].data_ptr(), v[i].data_ptr()
            c.k_scale, c.v_scale = k_scale[i].data_ptr(), v_scale[i].data_ptr()
            c.block_table, c.lengths = block_table.data_ptr(), lengths.data_ptr()
            c.status = self._status.data_ptr()
            c.num_pages, c.page_size, c.kv_heads, c.head_dim = pages, page, heads, hd
            c.batch, c.table_columns, c.format = batch, columns, _lib.KV_FORMATS[fmt]
            # an empty write makes every check of the shape and touches nothing
            _lib.check(self._lib.tt_kv_write(ctypes.byref(c), 0, None, None, None, None, 0, None,
                                             None), "KVCache", self._lib)

    # ---- lengths ------------------------------------------------------------
    def advance(self, tokens: int, new_tokens: Optional[torch.Tensor] = None) -> None:
        """Add `tokens` new tokens to every sequence, or new_tokens[b], at most
        `tokens` and not negative, to sequence b. Refuses what `max_tokens` has
        no room for. As long as `advance` and `reset` alone change the lengths, the
        host keeps a bound on them, and reads them from the device only near
        `max_tokens`. Once anything else has written into `lengths`, a graph with it
        or with an `advance` in it was captured, or `lengths_changed` was called,
        and in a cache over the caller's tensors, every call reads them, as a
        replay may change them unseen. (While a CUDA graph is captured, and in its
        replays, the host cannot know the lengths; one beyond the room is then
        latched on the device.)"""
        if tokens < 0:
            raise ValueError("tokens must be >= 0")
        new_tokens = self._counts(new_tokens)
        known = self._bound_holds()
        if not torch.cuda.is_current_stream_capturing():
            if not known or self._longest + tokens > self.max_tokens:
                grown = self.lengths + (tokens if new_tokens is None else new_tokens)
                longest = int(grown.max()) if self.batch else 0
                if longest > self.max_tokens:
                    raise ValueError(f"cache is full: a sequence would hold {longest} tokens of "
                                     f"at most {self.max_tokens}")
                self._longest = longest
            else:
                self._longest += tokens
        else:
            self._seen = None
        self.lengths.add_(tokens if new_tokens is None else new_tokens)
        if self._seen is not None:
            self._seen = self.lengths._version

    def reset(self) -> None:
        """Forget every token (lengths 0); the pages stay where they are."""
        known = self._bound_holds() and not torch.cuda.is_current_stream_capturing()
        self.lengths.zero_()
        self._longest, self._seen = 0, self.lengths._version if known else None

    def lengths_changed(self) -> None:
        """Say that `lengths` changes by means that torch does not count (kernels of the
        caller's own, `.data`): from now on `advance` reads it on every call."""
        self._seen = None

    def _bound_holds(self) -> bool:
        if self._seen is not None and self._seen != self.lengths._version:
            self._seen = None
        return self._seen is not None

    # ---- the operators ------------------------------------------------------
    # What a call's shapes, strides and types decide (its checks, the constant
    # arguments of the C call) is worked out once and kept under those; a step's
    # call then costs little more than its launches.
    def write(self, k: torch.Tensor, v: torch.Tensor, new_tokens: Optional[torch.Tensor] = None,
              layer: int = 0) -> None:
        """Quantise the keys and values of new tokens into layer `layer`: k and
        v are [batch, tokens, kv_heads, head_dim] float32, float16 or bfloat16
        (any strides with head_dim contiguous). new_tokens, [batch] int32, says
        how many leading rows of each sequence are new tokens (default: all);
        `lengths` counts them already."""
        key = (layer, k.shape, k.stride(), k.dtype, k.get_device(), v.shape, v.stride(), v.dtype,
               v.get_device())
        plan = self._plans.get(key)
        if plan is None:
            for name, t in (("k", k), ("v", v)):
                self._check(t, name, self.kv_heads)
            if k.shape != v.shape or k.dtype != v.dtype:
                raise ValueError(f"k and v must agree in shape and type, got {tuple(k.shape)} "
                                 f"{k.dtype} and {tuple(v.shape)} {v.dtype}")
            if k.stride(3) != 1 or v.stride(3) != 1:
                return self.write(k.contiguous(), v.contiguous(), new_tokens, layer)
            plan = self._keep(key, (self._struct(layer), _dtype_code(k, "k"), _strides(k),
                                    _strides(v), k.shape[1]))
        struct, dtype, ks, vs, n = plan
        counts = None if new_tokens is None else self._counts(new_tokens)
        if _current_device() != self._index:
            with torch.cuda.device(self.device):
                return self.write(k, v, new_tokens, layer)
        rc = self._c_write(struct, dtype, k.data_ptr(), v.data_ptr(), ks, vs, n,
                           None if counts is None else counts.data_ptr(), _raw_stream(self._index))
        if rc != 0:
            _lib.check(rc, "tt_kv_write", self._lib)

    def read(self, dtype: torch.dtype = torch.float32, max_tokens: Optional[int] = None,
             layer: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
        """The first max_tokens (default: as many as there is room for) tokens
        of every sequence in layer `layer`: k and v, [batch, max_tokens,
        kv_heads, head_dim] of `dtype`, zero behind each sequence's end."""
        n = self.max_tokens if max_tokens is None else max_tokens
        if n < 0:
            raise ValueError("max_tokens must be >= 0")
        struct = self._struct(layer)
        shape = (self.batch, n, self.kv_heads, self.head_dim)
        k = torch.empty(shape, dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        if _current_device() != self._index:
            with torch.cuda.device(self.device):
                return self.read(dtype, max_tokens, layer)
        rc = self._c_read(struct, _dtype_code(k, "dtype"), k.data_ptr(), v.data_ptr(), n,
                          _raw_stream(self._index))
        if rc != 0:
            _lib.check(rc, "tt_kv_read", self._lib)
        return k, v

    def attend(self, q: torch.Tensor, new_tokens: Optional[torch.Tensor] = None, layer: int = 0,
               scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Causal attention of the new tokens over layer `layer`, which holds
        their keys and values already. q is [batch, tokens, heads, head_dim]
        (strides as in `write`), heads a multiple of kv_heads: query head h
        reads key head h // (heads // kv_heads). Row i < new_tokens[b] stands at
        position lengths[b] - new_tokens[b] + i and sees the tokens up to its
        own. `scale` (default head_dim ** -0.5; positive) multiplies the scores. Returns
        (or writes to `out`, contiguous, sharing no memory with q) [batch,
        tokens, heads, head_dim] of q's type, computed to fp32 accuracy and
        rounded once; rows behind new_tokens[b] are 0."""
        key = (layer, q.shape, q.stride(), q.dtype, q.get_device())
        plan = self._plans.get(key)
        if plan is None:
            if q.dim() != 4 or q.shape[2] % self.kv_heads or q.shape[2] == 0:
                raise ValueError(f"q must be [batch, tokens, heads, head_dim] with heads a multiple "
                                 f"of {self.kv_heads}, got {tuple(q.shape)}")
            self._check(q, "q", q.shape[2])
            if q.stride(3) != 1:
                return self.attend(q.contiguous(), new_tokens, layer, scale, out)
            dtype = _dtype_code(q, "q")
            with torch.cuda.device(self.device):
                nbytes = self._lib.tt_kv_attention_typed_workspace_bytes(self._structs[0], dtype,
                                                                         q.shape[1], q.shape[2])
            plan = self._keep(key, (self._struct(layer), dtype, _strides(q), q.shape[1],
                                    q.shape[2], nbytes))
        struct, dtype, strides, n, heads, nbytes = plan
        counts = None if new_tokens is None else self._counts(new_tokens)
        if _current_device() != self._index:
            with torch.cuda.device(self.device):
                return self.attend(q, new_tokens, layer, scale, out)
        if out is None:
            out = q.new_empty(q.shape)
        elif (out.shape != q.shape or out.dtype != q.dtype or out.device != q.device
              or not out.is_contiguous()):
            raise ValueError("out must be a contiguous tensor of q's shape, type and device")
        ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device) if nbytes else None
        rc = self._c_attend(struct, dtype, q.data_ptr(), strides, n, heads,
                            None if counts is None else counts.data_ptr(),
                            self._scale if scale is None else scale, out.data_ptr(),
                            None if ws is None else ws.data_ptr(), nbytes, _raw_stream(self._index))
        if rc != 0:
            _lib.check(rc, "tt_kv_attention", self._lib)
        return out

    def read_device_status(self) -> Tuple[int, int]:
        """Synchronise, return and clear (code, detail) latched by the kernels' checks
        of lengths, counts, block-table entries and scales; (0, 0) when all were in range."""
        if _current_device() != self._index:  # a default stream is the current device's
            with torch.cuda.device(self.device):
                return self.read_device_status()
        code, detail = ctypes.c_int32(0), ctypes.c_int32(0)
        stream = _raw_stream(self._index)
        _lib.check(self._lib.tt_kv_read_status(self._structs[0], ctypes.byref(code),
                                               ctypes.byref(detail), stream),
                   "tt_kv_read_status", self._lib)
        return code.value, detail.value

    # ---- checks -------------------------------------------------------------
    def _check(self, t: torch.Tensor, name: str, heads: int) -> None:
        if not t.is_cuda:
            raise RuntimeError("KVCache runs on CUDA only (no CPU path)")
        if t.device != self.device:
            raise ValueError(f"{name} must be on {self.device}, got {t.device}")
        if t.dim() != 4 or t.shape[0] != self.batch or t.shape[2] != heads or \
                t.shape[3] != self.head_dim:
            raise ValueError(f"{name} must be [{self.batch}, tokens, {heads}, {self.head_dim}], "
                             f"got {tuple(t.shape)}")

    def _struct(self, layer: int):
        if not 0 <= layer < self.num_layers:
            raise ValueError(f"layer must be in [0, {self.num_layers}), got {layer}")
        return self._structs[layer]

    def _keep(self, key, plan):
        if len(self._plans) >= 1024:  # prompts of ever new lengths
            self._plans.clear()
        self._plans[key] = plan
        return plan

    def _counts(self, new_tokens: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
        if new_tokens is None:
            return None
        if (new_tokens.shape != (self.batch,) or new_tokens.dtype != torch.int32
                or new_tokens.get_device() != self._index):
            raise ValueError(f"new_tokens must be an int32 tensor of shape ({self.batch},) on "
                             f"{self.device}, got {new_tokens.dtype} of "
                             f"{tuple(new_tokens.shape)} on {new_tokens.device}")
        return new_tokens if new_tokens.is_contiguous() else new_tokens.contiguous()


def _strides(t: torch.Tensor):
    s = t.stride()
    return (ctypes.c_int64 * 3)(s[0], s[1], s[2])


# The current device and stream without the Python objects that torch.cuda makes
# of them, where this torch has the functions behind it.
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _stream_of(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or _stream_of
