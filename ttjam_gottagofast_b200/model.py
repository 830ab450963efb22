"""Drop-in `UserOptimizedTransformer` on the sm_100a kernels.

The module mirrors the reference contract (torch_transformer_benchmark.py):

* constructor `UserOptimizedTransformer(config)` with a `TransformerConfig`
  (:149-160, :175);
* the same submodules in the same construction order -- `layers.{i}.norm1`,
  `layers.{i}.attention.{q,k,v,out}_proj`, `layers.{i}.norm2`,
  `layers.{i}.ffn_in`, `layers.{i}.ffn_out`, `final_norm` (:72-75, :128-132,
  :152-160) -- so `load_state_dict(strict=True)` / `copy_model_weights`
  (:203-213) work unchanged and `torch.manual_seed(s)` draws identical weights;
* `forward(x, valid_token_mask=None)` -> [B, S, d_model] (:185-199).

The contract declares `class UserOptimizedTransformer(BaselineTransformer)`
(:175). `derive_user_optimized(BaselineTransformer)` builds exactly that class
from the caller's own base; the stand-alone `UserOptimizedTransformer` here
holds the same parameters in classes of its own, for callers without the
reference module. Both run the forward below.

The forward is CUDA only. It packs the parameters into a device image on first
use and again whenever they change: `load_state_dict`, `.to()`, or an
in-place write through an autograd-visible op (tensor version counters). A
write through `.data`, or replacing a Parameter object, is invisible to those
counters: call `invalidate()` after one. The output and the scratch come from
PyTorch's caching allocator, and the kernels run on
`torch.cuda.current_stream()` without a host sync. There is no CPU path: a CPU
input raises.

Parameters and inputs may be float32, float16 or bfloat16 (the reference's
`--dtype`, :225-231, moves model and input to one of them). The parameters
share one dtype; the input's may differ; the output has the input's dtype.
16-bit values widen exactly to fp32 and every schedule computes in fp32
accuracy; a 16-bit output is that result rounded once to nearest even.

`forward_cached(x, cache)` runs a causal model on new tokens alone, over an
8-bit key/value cache (`make_cache`, kv_cache.py) of the earlier ones.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch
import torch.nn as nn

from . import _lib
from .kv_cache import KVCache


class SelfAttention(nn.Module):
    """Parameter holder with BaselineSelfAttention's names (:62-75)."""

    def __init__(self, d_model: int, num_heads: int) -> None:
        super().__init__()
        if d_model % num_heads != 0:
            raise ValueError("d_model must be divisible by num_heads")
        self.d_model = d_model
        self.num_heads = num_heads
        self.head_dim = d_model // num_heads
        self.scale = self.head_dim ** -0.5
        self.q_proj = nn.Linear(d_model, d_model, bias=True)
        self.k_proj = nn.Linear(d_model, d_model, bias=True)
        self.v_proj = nn.Linear(d_model, d_model, bias=True)
        self.out_proj = nn.Linear(d_model, d_model, bias=True)


class TransformerBlock(nn.Module):
    """Parameter holder with BaselineTransformerBlock's names (:125-132)."""

    def __init__(self, d_model: int, num_heads: int, ffn_dim: int) -> None:
        super().__init__()
        self.norm1 = nn.LayerNorm(d_model)
        self.attention = SelfAttention(d_model, num_heads)
        self.norm2 = nn.LayerNorm(d_model)
        self.ffn_in = nn.Linear(d_model, ffn_dim)
        self.ffn_out = nn.Linear(ffn_dim, d_model)


class TTForward:
    """The forward pass on libttjam_b200.so, for any nn.Module that holds the
    reference's parameters under the reference's names (`layers.{i}...`,
    `final_norm`) and its config as `self.config`."""

    def _tt_setup(self, config) -> None:
        config.validate()
        self._lib = _lib.load()
        self._plan = "auto"
        self._flags = 0
        self._cfg = _lib.make_config(config)
        _lib.check(self._lib.tt_validate_config(ctypes.byref(self._cfg)), "config")
        self._image: Optional[torch.Tensor] = None
        self._image_key = None
        self._plist = None
        self._ws_bytes = {}
        self._host_inflight = []  # (event, host buffers) of tt_forward_host calls in flight
        self._host_events = []    # events of finished entries, for reuse
        self.fp16_operand_bound = None
        self.register_load_state_dict_post_hook(
            lambda module, incompatible: module.invalidate())

    # ---- packed image -----------------------------------------------------
    def set_plan(self, plan: str = "auto") -> None:
        """Force a kernel schedule ("auto", "cluster", "ops_ffma", "ops_tc")
        for tests and measurements; "auto" picks the fastest applicable one."""
        cfg = _lib.make_config(self.config, plan, self._flags)
        _lib.check(self._lib.tt_validate_config(ctypes.byref(cfg)), "plan")
        self._plan = plan
        self._cfg = cfg
        self._ws_bytes = {}

    def _set_flags(self, flags: int) -> None:
        if flags != self._flags:
            self._flags = flags
            self._cfg = _lib.make_config(self.config, self._plan, flags)
            self._ws_bytes = {}

    def invalidate(self) -> None:
        """Drop the packed device image; the next forward repacks it."""
        self._image = None
        self._image_key = None
        self._plist = None

    def _apply(self, fn, *args, **kwargs):
        self.invalidate()
        return super()._apply(fn, *args, **kwargs)

    def _param_key(self):
        # Version counters only grow, so their sum changes with any in-place
        # write to any parameter; the parameter objects are fixed between
        # invalidations (load_state_dict and .to() invalidate).
        plist = self._plist
        if plist is None:
            plist = self._plist = tuple(self.parameters())
        return sum(p._version for p in plist)

    def _ensure_image(self, device: torch.device) -> torch.Tensor:
        key = self._param_key()
        image = self._image
        if image is not None and key == self._image_key and image.device == device:
            return image
        self._plist = None
        key = self._param_key()
        # float32, float16 or bfloat16 parameters, all of one dtype (the
        # reference's --dtype moves the whole model, :698-699); 16-bit ones
        # widen exactly to fp32 as they are packed
        pdtype = next(self.parameters()).dtype
        for name, p in self.named_parameters():
            if (p.device != device or p.dtype != pdtype or not p.is_contiguous()
                    or str(p.dtype).split(".")[-1] not in _lib.DTYPE_CODES):
                raise ValueError(f"parameter {name} must be a contiguous float32, float16 or "
                                 f"bfloat16 tensor on {device}, all parameters of one dtype "
                                 f"(got {p.dtype} on {p.device}; the first is {pdtype})")
        dcode = _lib.DTYPE_CODES[str(pdtype).split(".")[-1]]
        lib = self._lib
        pcfg = _lib.make_config(self.config)
        nbytes = lib.tt_image_bytes(ctypes.byref(pcfg))
        image = torch.empty(nbytes, dtype=torch.uint8, device=device)
        arr = (_lib.TTLayerParams * len(self.layers))()
        for i, blk in enumerate(self.layers):
            a = blk.attention
            ptrs = dict(
                norm1_weight=blk.norm1.weight, norm1_bias=blk.norm1.bias,
                q_weight=a.q_proj.weight, q_bias=a.q_proj.bias,
                k_weight=a.k_proj.weight, k_bias=a.k_proj.bias,
                v_weight=a.v_proj.weight, v_bias=a.v_proj.bias,
                out_weight=a.out_proj.weight, out_bias=a.out_proj.bias,
                norm2_weight=blk.norm2.weight, norm2_bias=blk.norm2.bias,
                ffn_in_weight=blk.ffn_in.weight, ffn_in_bias=blk.ffn_in.bias,
                ffn_out_weight=blk.ffn_out.weight, ffn_out_bias=blk.ffn_out.bias)
            for field, t in ptrs.items():
                setattr(arr[i], field, t.data_ptr())
        stream = torch.cuda.current_stream(device).cuda_stream
        _lib.check(lib.tt_pack_image_typed(ctypes.byref(pcfg), dcode, arr,
                                           self.final_norm.weight.data_ptr(),
                                           self.final_norm.bias.data_ptr(), image.data_ptr(),
                                           nbytes, stream), "tt_pack_image", lib)
        # The split-precision schedule holds activations as fp16 pieces; when
        # the weights allow one beyond the fp16 range for some input, the
        # automatic plan keeps to the fp32 schedules (set-up time: this syncs).
        bound = ctypes.c_float(0.0)
        _lib.check(lib.tt_fp16_operand_bound(ctypes.byref(pcfg), image.data_ptr(),
                                             ctypes.byref(bound), stream),
                   "tt_fp16_operand_bound", lib)
        self.fp16_operand_bound = bound.value
        safe = bound.value < _lib.TT_FP16_MAX  # False for inf and NaN too
        self._set_flags(0 if safe else _lib.TT_FLAG_FP32_ONLY)
        self._image = image
        self._image_key = key
        return image

    # ---- forward ----------------------------------------------------------
    def forward(self, x: torch.Tensor,
                valid_token_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        if not x.is_cuda:
            raise RuntimeError("UserOptimizedTransformer runs on CUDA only (no CPU path)")
        dname = str(x.dtype).split(".")[-1]
        if dname not in _lib.DTYPE_CODES:
            raise ValueError(f"expected a float32, float16 or bfloat16 input, got {x.dtype}")
        dcode = _lib.DTYPE_CODES[dname]
        if x.dim() != 3 or x.shape[-1] != self.config.d_model:
            raise ValueError(f"expected x of shape [B, S, {self.config.d_model}], "
                             f"got {tuple(x.shape)}")
        if not x.is_contiguous() or x.data_ptr() % 16:
            x = x.contiguous().clone() if x.data_ptr() % 16 else x.contiguous()
        b, s, _ = x.shape
        mask_ptr = None
        if valid_token_mask is not None:
            m = valid_token_mask
            if m.shape != (b, s):
                raise ValueError(f"valid_token_mask must be [B, S] = {(b, s)}, got "
                                 f"{tuple(m.shape)}")
            if m.device != x.device:
                raise ValueError("valid_token_mask must be on the same device as x")
            if m.dtype != torch.bool and m.dtype != torch.uint8:
                raise ValueError(f"valid_token_mask must be bool, got {m.dtype}")
            if not m.is_contiguous():
                m = m.contiguous()
            valid_token_mask = m
            mask_ptr = m.data_ptr()
        device = x.device
        image = self._ensure_image(device)
        lib, cfg = self._lib, self._cfg
        y = torch.empty_like(x)
        ws_bytes = self._ws_bytes.get((b, s, dcode))
        if ws_bytes is None:
            ws_bytes = self._ws_bytes[(b, s, dcode)] = lib.tt_typed_workspace_bytes(
                ctypes.byref(cfg), dcode, b, s)
        ws_ptr = None
        if ws_bytes:
            ws = torch.empty(ws_bytes, dtype=torch.uint8, device=device)
            ws_ptr = ws.data_ptr()
        stream = torch.cuda.current_stream(device).cuda_stream
        if dcode == _lib.TT_DTYPE_F32:
            rc = lib.tt_forward(ctypes.byref(cfg), image.data_ptr(), x.data_ptr(), mask_ptr, b,
                                s, y.data_ptr(), ws_ptr, ws_bytes, stream)
        else:
            # 16-bit x and y: widened to fp32, the fp32 schedule, rounded back
            rc = lib.tt_forward_typed(ctypes.byref(cfg), image.data_ptr(), dcode, x.data_ptr(),
                                      mask_ptr, b, s, y.data_ptr(), ws_ptr, ws_bytes, stream)
        if rc != 0:
            _lib.check(rc, "tt_forward", lib)
        return y

    def forward_host(self, x_host: torch.Tensor, valid_token_mask: Optional[torch.Tensor] = None,
                     out: Optional[torch.Tensor] = None, device=None,
                     slices: Optional[int] = None) -> torch.Tensor:
        """The forward pass from host buffers to host buffers, with the copies
        overlapped with the compute: the batch runs as `slices` consecutive
        slices of whole sequences (sequences are independent); slice i+1's
        inputs cross to the device on one copy stream while slice i computes on
        the current stream, and slice i's output crosses back on another
        while slice i+1 computes. Pinned host buffers make the copies
        asynchronous (pageable ones still give correct results, without the
        overlap). A call small enough for one slice is one library call
        (tt_forward_host: copy in, forward, copy out).

        `x_host` is [B, S, d_model] float32 on the CPU, `valid_token_mask`
        [B, S] bool on the CPU or None, `out` an optional [B, S, d_model]
        float32 CPU tensor to write (allocated pinned when omitted). Returns
        `out`. Like a non_blocking copy, the call returns once the work is
        enqueued: the current stream of `device` (default: the current CUDA
        device) has the whole forward and the last copy ordered before
        anything enqueued on it later, so synchronise that stream before
        reading `out`."""
        if x_host.is_cuda:
            raise ValueError("forward_host takes host buffers; call the module for device tensors")
        if x_host.dtype != torch.float32 or x_host.dim() != 3:
            raise ValueError("expected a float32 [B, S, d_model] host tensor")
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None else \
            torch.device(device)
        if dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        b, s, d = x_host.shape
        if out is None:
            out = torch.empty((b, s, d), dtype=torch.float32, pin_memory=True)
        if out.shape != x_host.shape or out.dtype != torch.float32 or out.is_cuda:
            raise ValueError("out must be a float32 host tensor shaped like x")
        if b == 0 or s == 0:
            return out
        if slices is None:
            # slices of at least 32768 tokens (smaller ones leave the GPU part
            # idle in each launch), at most 8: only the first slice's copy in
            # and the last one's copy out are not hidden
            slices = min(8, b, max(1, (b * s) // 32768))
        slices = max(1, min(slices, b))
        cur = torch.cuda.current_stream(dev)
        if slices == 1:
            self._host_step(x_host, valid_token_mask, out, dev)
            return out
        cin = torch.cuda.Stream(dev)
        cout = torch.cuda.Stream(dev)
        x_dev = torch.empty((b, s, d), dtype=torch.float32, device=dev)
        m_dev = (None if valid_token_mask is None else
                 torch.empty((b, s), dtype=valid_token_mask.dtype, device=dev))
        cin.wait_stream(cur)   # the buffers come from the current stream's pool
        cout.wait_stream(cur)
        bounds = self._slice_bounds(b, slices)
        for i in range(slices):
            lo, hi = bounds[i], bounds[i + 1]
            if lo == hi:
                continue
            with torch.cuda.stream(cin):
                x_dev[lo:hi].copy_(x_host[lo:hi], non_blocking=True)
                if m_dev is not None:
                    m_dev[lo:hi].copy_(valid_token_mask[lo:hi], non_blocking=True)
            cur.wait_stream(cin)
            y = self.forward(x_dev[lo:hi], None if m_dev is None else m_dev[lo:hi])
            cout.wait_stream(cur)
            with torch.cuda.stream(cout):
                out[lo:hi].copy_(y, non_blocking=True)
            y.record_stream(cout)
        cur.wait_stream(cout)
        x_dev.record_stream(cin)
        if m_dev is not None:
            m_dev.record_stream(cin)
        return out

    def _host_step(self, x_host, mask, out, dev) -> None:
        """One small host-buffer step as one library call (tt_forward_host):
        the copy in, the forward and the copy out are enqueued in C, so the
        per-call host work that limits small steps is a single entry."""
        b, s, _ = x_host.shape
        if mask is not None:
            if mask.shape != (b, s) or mask.dtype not in (torch.bool, torch.uint8):
                raise ValueError(f"valid_token_mask must be a bool [B, S] = {(b, s)} tensor")
            if not mask.is_contiguous():
                mask = mask.contiguous()
            # an all-true mask computes exactly what no mask computes: skip its
            # copy (one of the three small copies that bound a small step)
            if mask.numel() <= (1 << 16) and bool(mask.all()):
                mask = None
        if not x_host.is_contiguous():
            x_host = x_host.contiguous()
        if dev.index != torch.cuda.current_device():
            with torch.cuda.device(dev):
                return self._host_step(x_host, mask, out, dev)
        image = self._ensure_image(dev)
        lib, cfg = self._lib, self._cfg
        key = (b, s, "host")
        nbytes = self._ws_bytes.get(key)
        if nbytes is None:
            nbytes = self._ws_bytes[key] = lib.tt_host_workspace_bytes(ctypes.byref(cfg), b, s)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        cur = torch.cuda.current_stream(dev)
        rc = lib.tt_forward_host(ctypes.byref(cfg), image.data_ptr(), x_host.data_ptr(),
                                 None if mask is None else mask.data_ptr(), b, s,
                                 out.data_ptr(), ws.data_ptr(), nbytes, cur.cuda_stream)
        if rc == 0:
            # the copies are asynchronous: keep the host buffers alive until the
            # stream has passed them, so a freed pinned block is not handed out
            # again (by torch's host allocator) while a copy still reads or
            # writes it; finished entries give their events back for reuse
            inflight, free = self._host_inflight, self._host_events
            while inflight and inflight[0][0].query():
                free.append(inflight.pop(0)[0])
            ev = free.pop() if free else torch.cuda.Event()
            ev.record(cur)
            inflight.append((ev, x_host, mask, out))
        if rc != 0:
            _lib.check(rc, "tt_forward_host", lib)

    @staticmethod
    def _slice_bounds(b: int, slices: int):
        """Sequence boundaries of the slices: with three or more, the first
        and the last are a quarter of the others (only the first one's copy
        in and the last one's copy out are not overlapped), the rest equal."""
        if slices < 3:
            return [b * i // slices for i in range(slices + 1)]
        edge = max(1, b // (4 * slices))
        inner = b - 2 * edge
        mids = [edge + inner * i // (slices - 2) for i in range(slices - 1)]
        return [0] + mids + [b]

    # ---- token by token ---------------------------------------------------
    def make_cache(self, batch: int, max_tokens: int, *, fmt: str = "e4m3",
                   page_size: int = 64, device=None) -> KVCache:
        """An empty 8-bit key/value cache for this model's layers, on the
        parameters' device unless told otherwise."""
        cfg = self.config
        if device is None:
            device = next(self.parameters()).device
        return KVCache(batch, max_tokens, cfg.num_heads, cfg.d_model // cfg.num_heads,
                       num_layers=cfg.num_layers, page_size=page_size, fmt=fmt, device=device)

    def forward_cached(self, x: torch.Tensor, cache: KVCache,
                       new_tokens: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The causal forward of new tokens alone: x [B, n, d_model] (float32,
        float16 or bfloat16) are the next n tokens of every sequence of
        `cache`, or the next new_tokens[b] <= n ([B] int32 on the device) of
        sequence b with padding behind them. Adds them to the cache (its
        lengths, and each layer's keys and values, rounded to 8 bits) and
        returns y [B, n, d_model] of x's type, zero at the padding. A prompt
        is one call, or several with pieces of it; a next token a call with
        n = 1. A call that raises once the arguments were accepted leaves the
        tokens counted in the cache."""
        if not x.is_cuda:
            raise RuntimeError("UserOptimizedTransformer runs on CUDA only (no CPU path)")
        dname = str(x.dtype).split(".")[-1]
        if dname not in _lib.DTYPE_CODES:
            raise ValueError(f"expected a float32, float16 or bfloat16 input, got {x.dtype}")
        dcode = _lib.DTYPE_CODES[dname]
        cfg = self.config
        if x.dim() != 3 or x.shape[0] != cache.batch or x.shape[-1] != cfg.d_model:
            raise ValueError(f"expected x of shape [{cache.batch}, n, {cfg.d_model}], "
                             f"got {tuple(x.shape)}")
        if x.device != cache.device:
            raise ValueError(f"cache must be on the same device as x, got {cache.device}")
        if not cfg.causal:
            raise ValueError("only a causal model runs token by token")
        if (cache.num_layers != cfg.num_layers or cache.kv_heads != cfg.num_heads
                or cache.head_dim * cfg.num_heads != cfg.d_model):
            raise ValueError("cache has other layers, heads or head_dim than the model")
        if x.device.index != torch.cuda.current_device():
            with torch.cuda.device(x.device):
                return self.forward_cached(x, cache, new_tokens)
        if not x.is_contiguous() or x.data_ptr() % 16:
            x = x.contiguous().clone() if x.data_ptr() % 16 else x.contiguous()
        b, n, _ = x.shape
        room = cache.block_table.shape[1] * cache.page_size
        if n > room:
            raise ValueError(f"{n} rows are more than a sequence has room for ({room} tokens)")
        counts = cache._counts(new_tokens)
        image = self._ensure_image(x.device)
        # a context averages values rounded to codes, which can exceed the
        # operand bound by 2^-4
        tight = self.fp16_operand_bound * 1.0625 >= _lib.TT_FP16_MAX
        ccfg = _lib.make_config(cfg, self._plan if self._plan.startswith("ops") else "auto",
                                _lib.TT_FLAG_FP32_ONLY if tight else self._flags)
        lib = self._lib
        y = torch.empty_like(x)
        nbytes = lib.tt_cached_workspace_bytes(ctypes.byref(ccfg), dcode, cache._array, b, n)
        if nbytes == 0 and x.numel():
            raise ValueError(f"tt_forward_cached: {_lib.last_error(lib)}")
        ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
        cache.advance(n, new_tokens=counts)
        stream = torch.cuda.current_stream(x.device).cuda_stream
        rc = lib.tt_forward_cached(ctypes.byref(ccfg), image.data_ptr(), dcode, x.data_ptr(),
                                   cache._array, None if counts is None else counts.data_ptr(), b, n,
                                   y.data_ptr(), ws.data_ptr(), nbytes, stream)
        if rc != 0:
            _lib.check(rc, "tt_forward_cached", lib)
        return y

    # ---- diagnostics ------------------------------------------------------
    def forward_plan(self, batch: int, seq: int) -> str:
        rc = self._lib.tt_forward_plan(ctypes.byref(self._cfg), batch, seq)
        if rc < 0:
            _lib.check(rc, "tt_forward_plan", self._lib)
        return _lib.PLAN_NAMES[rc]

    def read_device_status(self):
        """Synchronise and return (code, detail) latched by the kernels; (0, 0)
        when every bounded device wait finished in time."""
        if self._image is None:
            return 0, 0
        code, detail = ctypes.c_int32(0), ctypes.c_int32(0)
        stream = torch.cuda.current_stream(self._image.device).cuda_stream
        _lib.check(self._lib.tt_read_status(ctypes.byref(self._cfg), self._image.data_ptr(),
                                            ctypes.byref(code), ctypes.byref(detail), stream),
                   "tt_read_status", self._lib)
        return code.value, detail.value


class UserOptimizedTransformer(TTForward, nn.Module):
    """The reference's drop-in hook (:175-200), backed by libttjam_b200.so,
    with parameter holders of its own (no reference import needed)."""

    def __init__(self, config) -> None:
        nn.Module.__init__(self)
        config.validate()
        self.config = config
        self.layers = nn.ModuleList([
            TransformerBlock(config.d_model, config.num_heads, config.ffn_dim)
            for _ in range(config.num_layers)])
        self.final_norm = nn.LayerNorm(config.d_model)
        self._tt_setup(config)


_DERIVED = {}


def derive_user_optimized(baseline_cls):
    """`class UserOptimizedTransformer(BaselineTransformer)` as the contract
    declares it (torch_transformer_benchmark.py:175): the caller's own
    `BaselineTransformer` builds the parameters (same modules, same seeded
    init) and this module's forward replaces its forward. One class per base."""
    cls = _DERIVED.get(baseline_cls)
    if cls is None:
        def __init__(self, config):
            baseline_cls.__init__(self, config)
            self._tt_setup(config)

        cls = type("UserOptimizedTransformer", (TTForward, baseline_cls),
                   {"__init__": __init__, "__doc__": UserOptimizedTransformer.__doc__,
                    "__module__": __name__})
        _DERIVED[baseline_cls] = cls
    return cls
