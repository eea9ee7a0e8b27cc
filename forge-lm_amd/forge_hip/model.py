"""Host-side mirror of the reference model and backend types over libforge_hip.

Names, argument meaning and error behaviour follow the reference:
  ModelConfig      src/LLM.Core/Model/ModelConfig.cs:8-25
  ModelPresets     src/LLM.Core/Model/ModelPresets.cs:23-58
  HipBackend       the CudaBackend sibling: device name / memory for the CLI banner
                   (src/LLM.Core/Tensor/Cuda/CudaBackend.cs:114-215, src/LLM.Cli/Program.cs:132-145)
  GptModel         ctor init from new Random(seed) (src/LLM.Core/Model/GptModel.cs:38-99),
                   ForwardLast (GptModel.cs:202-209), parameter registry (Parameters.cs:29-58)
  BackendSelection src/LLM.Core/Tensor/BackendSelection.cs:13-34 plus the "hip" name
  TrainingRandom   PCG32, src/LLM.Core/Training/TrainingRandom.cs:13-72 (synthetic prompts)
"""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass
from typing import Callable, Optional, Sequence

import numpy as np

from . import _native as N


@dataclass(frozen=True)
class ModelConfig:
    vocab_size: int
    context_length: int
    d_model: int
    n_layers: int
    n_heads: int

    def __post_init__(self):
        if self.vocab_size <= 0:
            raise ValueError("VocabSize must be positive.")
        if self.context_length <= 0:
            raise ValueError("ContextLength must be positive.")
        if self.d_model <= 0:
            raise ValueError("DModel must be positive.")
        if self.n_layers <= 0:
            raise ValueError("NLayers must be positive.")
        if self.n_heads <= 0:
            raise ValueError("NHeads must be positive.")
        if self.d_model % self.n_heads != 0:
            raise ValueError(f"DModel ({self.d_model}) must be divisible by NHeads ({self.n_heads}).")

    @property
    def head_dim(self) -> int:
        return self.d_model // self.n_heads

    @property
    def mlp_hidden(self) -> int:
        return 4 * self.d_model

    def parameter_count(self) -> int:
        """VD + CD + L(12D^2 + 13D) + 2D (ModelPresets.cs:49-58)."""
        d = self.d_model
        return (self.vocab_size * d + self.context_length * d
                + self.n_layers * (12 * d * d + 13 * d) + 2 * d)


@dataclass(frozen=True)
class ModelPreset:
    key: str
    model_name: str
    context_length: int
    d_model: int
    layers: int
    heads: int

    def create_config(self, vocab_size: int) -> ModelConfig:
        return ModelConfig(vocab_size, self.context_length, self.d_model, self.layers, self.heads)

    def parameter_count(self, vocab_size: int) -> int:
        return self.create_config(vocab_size).parameter_count()


PRESETS = (
    ModelPreset("forge-98m", "Forge-98M", 512, 768, 12, 12),
    ModelPreset("forge-220m", "Forge-220M", 1024, 1024, 16, 16),
    ModelPreset("forge-320m", "Forge-320M", 1024, 1024, 24, 16),
)


def get_preset(key: str) -> ModelPreset:
    for p in PRESETS:
        if p.key.lower() == key.lower():
            return p
    raise ValueError(f"Unknown model preset '{key}'. Expected {', '.join(p.key for p in PRESETS)}, or custom.")


class TrainingRandom:
    """PCG32 (TrainingRandom.cs:13-72); used for the synthetic prompt ids."""
    _MUL = 6364136223846793005
    _M64 = (1 << 64) - 1

    def __init__(self, seed: int):
        self._inc = 0xDA3E39CB94B95BDB
        self._state = 0
        self._next_u32()
        self._state = (self._state + (seed & 0xFFFFFFFF)) & self._M64
        self._next_u32()

    def _next_u32(self) -> int:
        old = self._state
        self._state = (old * self._MUL + self._inc) & self._M64
        xs = (((old >> 18) ^ old) >> 27) & 0xFFFFFFFF
        rot = old >> 59
        return ((xs >> rot) | (xs << ((-rot) & 31))) & 0xFFFFFFFF

    def next(self, max_exclusive: int) -> int:
        if max_exclusive <= 0:
            raise ValueError("Upper bound must be positive.")
        bound = max_exclusive
        threshold = ((1 << 32) - bound) % bound
        while True:
            v = self._next_u32()
            if v >= threshold:
                return v % bound

    def ids(self, max_exclusive: int, n: int) -> np.ndarray:
        return np.array([self.next(max_exclusive) for _ in range(n)], dtype=np.int32)


class Random:
    """new System.Random(seed) NextDouble() stream, generated by the library."""

    def __init__(self, seed: int):
        self.seed = int(seed)
        self._pos = 0
        self._buf = np.empty(0, np.float64)

    def _ensure(self, n: int):
        if n > self._buf.size:
            size = max(n, 2 * self._buf.size, 1024)
            out = np.empty(size, np.float64)
            N.check(N.lib().fh_random_doubles(self.seed, size, out.ctypes.data))
            self._buf = out

    def next_double(self) -> float:
        self._ensure(self._pos + 1)
        v = float(self._buf[self._pos])
        self._pos += 1
        return v

    def next_doubles(self, n: int) -> np.ndarray:
        v = self.peek_doubles(n)
        self._pos += n
        return v

    def peek_doubles(self, n: int) -> np.ndarray:
        """The next n NextDouble values without consuming them."""
        self._ensure(self._pos + n)
        return self._buf[self._pos:self._pos + n].copy()

    def skip(self, n: int) -> None:
        """Consumes n values (the steps a generation actually sampled)."""
        self._ensure(self._pos + n)
        self._pos += n


def _dtype(name: str) -> int:
    return {"f32": N.FH_DTYPE_F32, "fp32": N.FH_DTYPE_F32, "bf16": N.FH_DTYPE_BF16}[name]


def _address(buf):
    """A DeviceBuffer's device address, or the address itself."""
    return buf.ptr if isinstance(buf, DeviceBuffer) else buf


def _room(*needs) -> None:
    """Checks the sizes of those of (name, buffer, bytes) that are DeviceBuffers."""
    for name, buf, nbytes in needs:
        if isinstance(buf, DeviceBuffer) and buf.nbytes < nbytes:
            raise ValueError(f"{name} needs {nbytes} bytes, the buffer has {buf.nbytes}")


@dataclass
class _Attention:
    qkv_cols: int
    out_cols: int
    kv: int
    scale: float
    dtype: int
    host: Optional[np.ndarray]

    @property
    def lengths(self):
        return None if self.host is None else self.host.ctypes.data


def _attention(qkv, out, lse, batch, T, n_heads, head_dim, n_kv_heads, lengths, scale, qkv_cols, out_cols, dtype,
               dout=None, dqkv=None) -> _Attention:
    """The defaults and the buffers' sizes of an attention call."""
    kv = n_heads if n_kv_heads is None else n_kv_heads
    qkv_cols = (n_heads + 2 * kv) * head_dim if qkv_cols is None else qkv_cols
    out_cols = n_heads * head_dim if out_cols is None else out_cols
    scale = (1.0 / math.sqrt(head_dim) if head_dim > 0 else 1.0) if scale is None else scale
    dt = _dtype(dtype)
    host = None
    if lengths is not None:
        host = np.ascontiguousarray(lengths, np.int32).reshape(-1)
        if host.size != batch:
            raise ValueError(f"{batch} lengths are needed, got {host.size}")
    rows, es = max(0, batch) * max(0, T), 2 if dt == N.FH_DTYPE_BF16 else 4
    wide = max(0, rows - 1) * es
    in_row, out_row = (n_heads + 2 * kv) * head_dim * es, n_heads * head_dim * es
    _room(("qkv", qkv, wide * qkv_cols + in_row), ("dqkv", dqkv, wide * qkv_cols + in_row),
          ("out", out, wide * out_cols + out_row), ("dout", dout, wide * out_cols + out_row),
          ("lse", lse, rows * max(0, n_heads) * 4))
    return _Attention(qkv_cols, out_cols, kv, float(scale), dt, host)


class HipBackend:
    """One device + stream (the `hip` backend behind ITensorBackend's selection)."""

    def __init__(self, device: int = 0):
        self._ctx = ctypes.c_void_p()
        N.check(N.lib().fh_context_create(device, ctypes.byref(self._ctx)))
        name = ctypes.create_string_buffer(256)
        mem = ctypes.c_uint64()
        cus = ctypes.c_int32()
        N.check(N.lib().fh_context_info(self._ctx, name, len(name), ctypes.byref(mem), ctypes.byref(cus)))
        self.device_name = name.value.decode()
        self.device_memory_bytes = mem.value
        self.compute_units = cus.value

    def memory(self) -> tuple:
        """(free device bytes, device bytes held as fh_sample_logits' scratch)."""
        fr, scr = ctypes.c_uint64(0), ctypes.c_uint64(0)
        N.check(N.lib().fh_context_memory(self._ctx, ctypes.byref(fr), ctypes.byref(scr)))
        return fr.value, scr.value

    @property
    def handle(self):
        return self._ctx

    def matmul_nn(self, a: "DeviceBuffer", b: "DeviceBuffer", y: "DeviceBuffer", M: int, K: int, N_: int,
                  accumulate: bool = False, dtype: str = "f32") -> None:
        """ITensorBackend.MatMulNN on device buffers (ITensorBackend.cs:22): y (+)= a @ b."""
        dt = {"f32": N.FH_DTYPE_F32, "fp32": N.FH_DTYPE_F32, "bf16": N.FH_DTYPE_BF16}[dtype]
        esz = 2 if dt == N.FH_DTYPE_BF16 else 4
        if a.nbytes < M * K * 4 or b.nbytes < K * N_ * esz or y.nbytes < M * N_ * 4:
            raise ValueError("buffer smaller than the product's operands")
        N.check(N.lib().fh_matmul_nn(self._ctx, a.ptr, b.ptr, y.ptr, M, K, N_, dt, int(bool(accumulate))))

    def attention_forward(self, qkv, out, lse, batch: int, T: int, n_heads: int, head_dim: int,
                          n_kv_heads: Optional[int] = None, lengths: Optional[Sequence[int]] = None,
                          scale: Optional[float] = None, qkv_cols: Optional[int] = None, out_cols: Optional[int] = None,
                          dtype: str = "f32") -> None:
        """Causal attention of packed q, k, v rows (fh_op_attention_forward): out rows and each row's log of
        its softmax sum (lse, fp32).  Buffers are DeviceBuffers or device addresses; scale defaults to
        1 / sqrt(head_dim), the widths to the packed ones, lengths to T each."""
        a = _attention(qkv, out, lse, batch, T, n_heads, head_dim, n_kv_heads, lengths, scale, qkv_cols, out_cols, dtype)
        N.check(N.lib().fh_op_attention_forward(self._ctx, _address(qkv), a.qkv_cols, _address(out), a.out_cols,
                                                _address(lse), a.lengths, batch, T, n_heads, a.kv, head_dim, a.scale,
                                                a.dtype))

    def attention_backward(self, dout, qkv, out, lse, dqkv, batch: int, T: int, n_heads: int, head_dim: int,
                           n_kv_heads: Optional[int] = None, lengths: Optional[Sequence[int]] = None,
                           scale: Optional[float] = None, qkv_cols: Optional[int] = None,
                           out_cols: Optional[int] = None, dtype: str = "f32") -> None:
        """The gradient dqkv of attention_forward's inputs from dout and its outputs (fh_op_attention_backward)."""
        a = _attention(qkv, out, lse, batch, T, n_heads, head_dim, n_kv_heads, lengths, scale, qkv_cols, out_cols, dtype,
                       dout, dqkv)
        N.check(N.lib().fh_op_attention_backward(self._ctx, _address(dout), _address(qkv), a.qkv_cols, _address(out),
                                                 a.out_cols, _address(lse), _address(dqkv), a.lengths, batch, T, n_heads,
                                                 a.kv, head_dim, a.scale, a.dtype))

    def distill_loss(self, logits, targets: Sequence[int], top_ids, top_logits, dlogits, T: int, V: int, K: int,
                     ignore_index: int = -1, temperature: float = 1.0, alpha: float = 1.0, dtype: str = "f32") -> float:
        """Mean distillation loss against a teacher's top logits and hard targets, and its gradient where
        dlogits is not None (fh_op_distill_loss).  Buffers are DeviceBuffers or device addresses: logits and
        dlogits [T, V] of dtype, top_ids [T, K] int32, top_logits [T, K] fp32."""
        dt = _dtype(dtype)
        tg = np.ascontiguousarray(targets, np.int32).reshape(-1)
        if tg.size < T:
            raise ValueError(f"{T} targets are needed, got {tg.size}")
        rows = max(0, T) * max(0, V) * (2 if dt == N.FH_DTYPE_BF16 else 4)
        _room(("logits", logits, rows), ("dlogits", dlogits, rows), ("top_ids", top_ids, max(0, T) * max(0, K) * 4),
              ("top_logits", top_logits, max(0, T) * max(0, K) * 4))
        loss = ctypes.c_float()
        N.check(N.lib().fh_op_distill_loss(self._ctx, _address(logits), tg.ctypes.data, _address(top_ids),
                                           _address(top_logits), None if dlogits is None else _address(dlogits), T, V, K,
                                           int(ignore_index), float(temperature), float(alpha), dt, ctypes.byref(loss)))
        return float(loss.value)

    def dispose(self):
        if self._ctx:
            N.lib().fh_context_destroy(self._ctx)
            self._ctx = ctypes.c_void_p()

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.dispose()

    def __del__(self):
        try:
            self.dispose()
        except Exception:
            pass


class DeviceBuffer:
    """A device allocation owned by a HipBackend (fh_buffer_*)."""

    def __init__(self, backend: HipBackend, nbytes: int):
        self.backend = backend
        self.nbytes = int(nbytes)
        self.ptr = ctypes.c_void_p()
        N.check(N.lib().fh_buffer_alloc(backend.handle, self.nbytes, ctypes.byref(self.ptr)))

    @classmethod
    def from_array(cls, backend: HipBackend, arr: np.ndarray) -> "DeviceBuffer":
        arr = np.ascontiguousarray(arr)
        buf = cls(backend, arr.nbytes)
        buf.write(arr)
        return buf

    def write(self, arr: np.ndarray) -> None:
        arr = np.ascontiguousarray(arr)
        if arr.nbytes > self.nbytes:
            raise ValueError("array larger than the buffer")
        N.check(N.lib().fh_buffer_write(self.backend.handle, self.ptr, arr.ctypes.data, arr.nbytes))

    def read(self, dtype, count: int) -> np.ndarray:
        out = np.empty(count, dtype)
        if out.nbytes > self.nbytes:
            raise ValueError("read larger than the buffer")
        N.check(N.lib().fh_buffer_read(self.backend.handle, out.ctypes.data, self.ptr, out.nbytes))
        return out

    def copy_from(self, src: "DeviceBuffer", nbytes: int | None = None) -> float:
        """ITensorBackend.Copy(src, self) on the device; returns the copy kernel's time in ms."""
        n = src.nbytes if nbytes is None else int(nbytes)
        if n > self.nbytes or n > src.nbytes:
            raise ValueError("copy larger than a buffer")
        ms = ctypes.c_float()
        N.check(N.lib().fh_buffer_copy(self.backend.handle, self.ptr, src.ptr, n, ctypes.byref(ms)))
        return float(ms.value)

    def checksum(self, nbytes: int | None = None) -> tuple:
        """(sum of the buffer's 32-bit words mod 2^64, ms of the pass that read it)."""
        n = self.nbytes if nbytes is None else int(nbytes)
        out, ms = ctypes.c_uint64(), ctypes.c_float()
        N.check(N.lib().fh_buffer_checksum(self.backend.handle, self.ptr, n, ctypes.byref(out), ctypes.byref(ms)))
        return int(out.value), float(ms.value)

    def free(self) -> None:
        if self.ptr:
            N.check(N.lib().fh_buffer_free(self.backend.handle, self.ptr))
            self.ptr = ctypes.c_void_p()


def _desc(cfg: ModelConfig, batch: int, dtype: str) -> N.ModelDesc:
    dt = {"f32": N.FH_DTYPE_F32, "fp32": N.FH_DTYPE_F32, "bf16": N.FH_DTYPE_BF16}[dtype]
    return N.ModelDesc(cfg.vocab_size, cfg.context_length, cfg.d_model, cfg.n_layers, cfg.n_heads, batch, dt, 0)


def registry(cfg: ModelConfig) -> list:
    """[(name, numel)] in registration order (GptModel.cs:53-91)."""
    desc = _desc(cfg, 1, "f32")
    out = []
    name = ctypes.create_string_buffer(128)
    numel = ctypes.c_int64()
    n = N.check(N.lib().fh_param_info(ctypes.byref(desc), 0, name, len(name), ctypes.byref(numel)))
    for i in range(n):
        N.check(N.lib().fh_param_info(ctypes.byref(desc), i, name, len(name), ctypes.byref(numel)))
        out.append((name.value.decode(), numel.value))
    return out


class GptModel:
    """Device-resident GPT session: weights + KV cache + history for `batch` sequences.

    ``GptModel(config, backend, seed)`` initialises like the reference ctor with
    ``new Random(seed)``; ``load_weights`` replaces them (registry order, fp32).
    ``dtype="bf16"`` stores matrices in bfloat16 (fp32 accumulation).
    """

    def __init__(self, config: ModelConfig, backend: HipBackend, seed: Optional[int] = None,
                 batch: int = 1, dtype: str = "f32", name: str = "Forge"):
        if not name.strip() or len(name) > 64:
            raise ValueError("Model name must contain 1-64 non-whitespace characters.")
        self.name = name
        self.config = config
        self.backend = backend
        self.batch = batch
        self.dtype = dtype
        self._desc = _desc(config, batch, dtype)
        self._s = ctypes.c_void_p()
        N.check(N.lib().fh_session_create(backend.handle, ctypes.byref(self._desc), ctypes.byref(self._s)))
        self._registry = registry(config)
        if seed is not None:
            N.check(N.lib().fh_session_init_random(self._s, int(seed)))

    @property
    def handle(self):
        return self._s

    @property
    def param_names(self) -> list:
        return [n for n, _ in self._registry]

    @property
    def param_count(self) -> int:
        return int(sum(n for _, n in self._registry))

    def load_weights(self, flat: np.ndarray) -> None:
        """Registry-order fp32 weights, flat (as Checkpoint.LoadCore reads them)."""
        flat = np.ascontiguousarray(flat, np.float32)
        if flat.size != self.param_count:
            raise ValueError(f"expected {self.param_count} floats, got {flat.size}")
        ptrs = (ctypes.c_void_p * len(self._registry))()
        o = 0
        for i, (_, n) in enumerate(self._registry):
            ptrs[i] = flat.ctypes.data + 4 * o
            o += n
        N.check(N.lib().fh_session_load_weights(self._s, ptrs, len(self._registry)))
        self._keep = flat

    def read_param(self, index_or_name) -> np.ndarray:
        idx = index_or_name if isinstance(index_or_name, int) else self.param_names.index(index_or_name)
        n = self._registry[idx][1]
        out = np.empty(n, np.float32)
        N.check(N.lib().fh_session_read_param(self._s, idx, out.ctypes.data, n))
        return out

    def read_weights(self) -> np.ndarray:
        return np.concatenate([self.read_param(i) for i in range(len(self._registry))])

    def forward_last(self, tokens) -> np.ndarray:
        """GptModel.ForwardLast: logits of the last row, [batch, V] (full recompute)."""
        ids = np.ascontiguousarray(tokens, np.int32)
        if ids.ndim == 1:
            ids = ids[None, :]
        out = np.empty((ids.shape[0], self.config.vocab_size), np.float32)
        N.check(N.lib().fh_forward_last(self._s, ids.ctypes.data, ids.shape[0], ids.shape[1], out.ctypes.data))
        return out

    def dispose(self):
        if self._s:
            N.lib().fh_session_destroy(self._s)
            self._s = ctypes.c_void_p()

    def __del__(self):
        try:
            self.dispose()
        except Exception:
            pass


class BackendSelection:
    """BackendSelection.Create (BackendSelection.cs:13-34) with `hip` added.

    Explicit names fail loudly; `auto` probes hip -> cuda -> cpu on Linux
    (hip -> cuda -> gpu -> cpu on Windows) and reports skipped candidates.
    """
    NAMES = ("auto", "cpu", "gpu", "cuda", "hip")

    @staticmethod
    def create(requested: str, is_windows: bool, factory: Callable[[str], object],
               on_unavailable: Optional[Callable[[str, Exception], None]] = None):
        name = requested.lower()
        if name not in BackendSelection.NAMES:
            raise ValueError(f"unknown backend '{requested}' (expected auto, cpu, gpu, cuda, or hip)")
        if name != "auto":
            return name, factory(name)
        candidates = ["hip", "cuda", "gpu", "cpu"] if is_windows else ["hip", "cuda", "cpu"]
        for c in candidates:
            try:
                return c, factory(c)
            except Exception as ex:  # noqa: BLE001 - mirrors the reference's catch-all for accelerators
                if c == "cpu":
                    raise
                if on_unavailable:
                    on_unavailable(c, ex)
        raise RuntimeError("CPU backend creation unexpectedly failed.")
