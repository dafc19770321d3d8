"""Host-side mirror of ferro's sampler interface over the gfx950 kernels.

- `SamplerParams` / `Sampler` mirror ferro::SamplerParams / ferro::Sampler (reference src/sampler.h:12-34): same
  field names, defaults and meaning; `Sampler.sample(logits, n_vocab, history)` returns the token id exactly as
  `int Sampler::sample(float*, int, const std::vector<int>&)` does, drawing from the same libstdc++ mt19937_64
  stream (one draw per non-greedy call, none for greedy: sampler.cpp:19-23, 45-46).
- `sample_batch`, `argmax_batch`, `verify` are the batched device entry points (fs_sample_batch, fs_argmax_batch,
  fs_verify) on torch CUDA tensors, launched on torch's current stream.
- `Edits` holds masks of allowed tokens and biases (fs_edits) for those calls and `decode_step`; `edit_batch` writes
  edited logits out, `logprobs` gives log-probabilities.

PyTorch only supplies device memory and streams; all sampling arithmetic runs in libferro_sampler.so.
"""
from __future__ import annotations

import ctypes
import threading
from collections.abc import Mapping
from dataclasses import dataclass

import numpy as np
import torch

from ._lib import FS_BF16, FS_F16, FS_F32, FS_MAX_TOP, PARAMS_DTYPE, FS_OK, FsEdits, SamplerError, check, lib

__all__ = ["SamplerParams", "Sampler", "Context", "Rng", "Edits", "params_array", "sample_batch", "argmax_batch", "verify",
           "edit_batch", "logprobs", "device_error", "PARAMS_DTYPE", "SamplerError"]

F32, BF16, F16 = FS_F32, FS_BF16, FS_F16          # types of logits (edit_batch, logprobs)


@dataclass
class SamplerParams:
    """ferro::SamplerParams (src/sampler.h:12-21) plus the frequency/presence extension (0 = off)."""
    temperature: float = 0.05
    top_k: int = 50
    top_p: float = 1.0
    min_p: float = 0.0
    repetition_penalty: float = 1.05
    repeat_last_n: int = -1
    penalty_from: int = 0
    seed: int = 0
    frequency_penalty: float = 0.0
    presence_penalty: float = 0.0
    softcap: float = 0.0              # > 0: the model's final-logit softcap, fused into the sampler's read

    def validate(self) -> None:
        """The server's range check (src/server.cpp:1071)."""
        if (self.temperature < 0 or self.top_p <= 0 or self.top_p > 1 or self.top_k < 0
                or self.repetition_penalty <= 0 or self.repeat_last_n < -1):
            raise ValueError("sampling parameter out of range")

    def is_greedy(self) -> bool:
        return np.float32(self.temperature) <= 0 or self.top_k == 1


def params_array(params) -> np.ndarray:
    """fs_row_params records from SamplerParams objects (or pass a PARAMS_DTYPE array through)."""
    if isinstance(params, np.ndarray) and params.dtype == PARAMS_DTYPE:
        return np.ascontiguousarray(params)
    if isinstance(params, SamplerParams):
        params = [params]
    out = np.zeros(len(params), PARAMS_DTYPE)
    for i, p in enumerate(params):
        out[i] = (p.temperature, p.top_k, p.top_p, p.min_p, p.repetition_penalty, p.frequency_penalty,
                  p.presence_penalty, p.repeat_last_n, p.penalty_from, p.softcap)
    return out


def _ptr(t):
    """Device pointer of a tensor the C ABI reads or writes as a packed array."""
    if t is None:
        return None
    if not t.is_contiguous():
        raise SamplerError("a non-contiguous tensor cannot be passed as a packed array")
    return ctypes.c_void_p(t.data_ptr())


def _lptr(t):
    """Device pointer of a logits matrix: rows may be strided (the C ABI takes the row stride ld), elements packed."""
    if t.dim() == 2 and t.shape[1] > 1 and t.stride(1) != 1:
        raise SamplerError("logits rows must be packed (stride 1 along the vocabulary)")
    return ctypes.c_void_p(t.data_ptr())


def _dev(x, dtype, device):
    """An input array or tensor as a packed device tensor of `dtype` (a strided view is copied, not misread)."""
    return torch.as_tensor(x, dtype=dtype, device=device).contiguous()


def _stream(stream=None):
    s = stream if stream is not None else torch.cuda.current_stream()
    return ctypes.c_void_p(s.cuda_stream)


def _hptr(a):
    """Host pointer of a numpy array (None: NULL)."""
    return None if a is None else a.ctypes.data_as(ctypes.c_void_p)


def _dev_params(params, device) -> torch.Tensor:
    if isinstance(params, torch.Tensor):
        if params.dtype != torch.uint8 or params.numel() % PARAMS_DTYPE.itemsize:
            raise SamplerError("params tensor must be uint8 bytes of fs_row_params records")
        return params.to(device).contiguous()
    a = params_array(params)
    return torch.from_numpy(a.view(np.uint8).copy()).to(device)


class Context:
    """An fs_context (device workspace); calls on one context are serialised by a lock."""

    _default = {}
    _dlock = threading.Lock()

    def __init__(self):
        h = ctypes.c_void_p()
        check(lib().fs_create(ctypes.byref(h)), "fs_create")
        self.h = h
        self.lock = threading.Lock()

    def __del__(self):
        h = getattr(self, "h", None)
        if h is not None and h.value:
            try:
                lib().fs_destroy(h)
            except Exception:
                pass

    def set_wait_limit(self, polls: int) -> None:
        """fs_set_wait_limit: the merge's bounded wait for a row's segments (0 = default)."""
        check(lib().fs_set_wait_limit(self.h, int(polls)), "fs_set_wait_limit")

    @classmethod
    def default(cls, device=None) -> "Context":
        dev = torch.device("cuda", torch.cuda.current_device() if device is None else torch.device(device).index or 0)
        with cls._dlock:
            if dev not in cls._default:
                cls._default[dev] = Context()
            return cls._default[dev]


class Rng:
    """fs_rng: libstdc++ std::mt19937_64 + generate_canonical, ferro::Sampler's draw stream (sampler.h:25,32)."""

    def __init__(self, seed: int = 0):
        h = ctypes.c_void_p()
        check(lib().fs_rng_create(ctypes.c_uint64(seed), ctypes.byref(h)), "fs_rng_create")
        self.h = h

    def __del__(self):
        h = getattr(self, "h", None)
        if h is not None and h.value:
            try:
                lib().fs_rng_destroy(h)
            except Exception:
                pass

    def next_u(self, n: int = 1) -> np.ndarray:
        out = np.zeros(n, np.float64)
        check(lib().fs_rng_next_u(self.h, out.ctypes.data_as(ctypes.c_void_p), n), "fs_rng_next_u")
        return out

    def copy(self) -> "Rng":
        r = Rng(1)
        check(lib().fs_rng_copy(self.h, r.h), "fs_rng_copy")
        return r


class DeviceRng:
    """fs_drng: one std::mt19937_64 draw stream per sampling stream, held on the device (ferro::Sampler's rng_,
    sampler.h:25,32). draw() gives each row of a sampling stream one generate_canonical draw, in row order; rows of
    greedy streams get 0 and consume nothing."""

    def __init__(self, seeds, device=None, stream=None):
        seeds = np.ascontiguousarray(np.asarray(seeds, dtype=np.uint64).reshape(-1))
        self.n = int(seeds.size)
        self._dev = torch.device("cuda" if device is None else device)
        h = ctypes.c_void_p()
        check(lib().fs_drng_create(self.n, seeds.ctypes.data_as(ctypes.c_void_p), _stream(stream),
                                   ctypes.byref(h)), "fs_drng_create")
        self.h = h

    def __del__(self):
        h = getattr(self, "h", None)
        if h is not None and h.value:
            try:
                lib().fs_drng_destroy(h)
            except Exception:
                pass

    def draw(self, params, row_off=None, peek=False, stream=None) -> torch.Tensor:
        p = _dev_params(params, self._dev)
        if p.numel() != self.n * PARAMS_DTYPE.itemsize:
            raise SamplerError("one params record per stream")
        ro = None
        rows = self.n
        if row_off is not None:
            ro = _dev(row_off, torch.int64, self._dev)
            if ro.numel() != self.n + 1:
                raise SamplerError("row_off must have n_streams+1 entries")
            rows = int(ro[-1].item())
        u = torch.empty(rows, dtype=torch.float64, device=self._dev)
        check(lib().fs_drng_draw(self.h, _ptr(ro), _ptr(p), _ptr(u), 1 if peek else 0, _stream(stream)),
              "fs_drng_draw")
        self._keep = (p, ro)
        return u

    def skip(self, counts, params, stream=None) -> None:
        p = _dev_params(params, self._dev)
        c = _dev(counts, torch.int32, self._dev)
        if c.numel() != self.n:
            raise SamplerError("one count per stream")
        check(lib().fs_drng_skip(self.h, _ptr(c), _ptr(p), _stream(stream)), "fs_drng_skip")
        self._keep = (p, c)

    def error(self, stream=None) -> int:
        bits = ctypes.c_int32(0)
        check(lib().fs_drng_error(self.h, _stream(stream), ctypes.byref(bits)), "fs_drng_error")
        return bits.value


def _check_logits(logits: torch.Tensor, V: int | None):
    if not (isinstance(logits, torch.Tensor) and logits.is_cuda and logits.dtype == torch.float32):
        raise SamplerError("logits must be a float32 CUDA tensor")
    if logits.dim() == 1:
        logits = logits.unsqueeze(0)
    if logits.dim() != 2:
        raise SamplerError("logits must be [B, V]")
    n = logits.shape[1] if V is None else V
    if n > logits.shape[1]:
        raise SamplerError("V exceeds the row length")
    ld = logits.stride(0) if logits.shape[0] > 1 else n + (-n) % 4
    if logits.stride(1) != 1 or ld % 4 or ld < n or logits.data_ptr() % 16:
        # the kernels take 16-byte aligned rows: repack into a padded copy
        padded = torch.zeros((logits.shape[0], n + (-n) % 4), dtype=torch.float32, device=logits.device)
        padded[:, :n] = logits[:, :n]
        logits, ld = padded, padded.stride(0)
    return logits, ld, n


def _hist_tensors(hist, hist_off, B, device):
    if hist is None:
        return None, None
    hist = _dev(hist, torch.int32, device)
    hist_off = _dev(hist_off, torch.int64, device)
    if hist_off.numel() != B + 1:
        raise SamplerError("hist_off must have B+1 entries")
    return hist, hist_off


# How sample_batch passes the parameters: "host" also hands the library their host copy (fs_sample_batch_hp, which
# picks the small-k kernel for batches it fits); "device" passes the device copy only (fs_sample_batch, the fused
# kernel for every batch). Tests run both.
ROUTE = "host"


class Edits:
    """Masks of allowed tokens and biases (fs_edits): what a program keeps from step to step for edits= of sample_batch,
    argmax_batch, verify, decode_step, edit_batch and logprobs.

    mask: int32 or uint32 words [n, W] (or [W]: one mask), W >= ceil(V / 32); token t is allowed where bit t % 32 of word
    t // 32 is set (as grammar engines write them; `pack` makes them from truth values). mask_of: each logits row's mask,
    negative: every token is allowed (default: row r takes mask r). bias: one {token: bias} per record, or CSR (ids,
    values, offsets) with ids ascending within a record; a record per row, per stream in verify. Arrays go to `device`
    here. Device tensors are read by each call, so a program may write the next step's masks into them: in place where
    they are packed int32 words (rows any stride apart), int32 mask_of and ids, float32 values and int64 offsets, else
    converted by every call."""

    def __init__(self, mask=None, mask_of=None, bias=None, device=None):
        dev = torch.device("cuda" if device is None else device)
        bias = None if bias is None else list(bias)
        if device is None:
            given = [mask, mask_of] + (bias or [])
            dev = next((t.device for t in given if isinstance(t, torch.Tensor) and t.is_cuda), dev)
        if dev.type == "cuda" and dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        self.device = dev
        self.mask = self.mask_of = self.bias_ids = self.bias = self.bias_off = None
        self._given = {}                                      # device tensors that each call converts
        if mask is not None:
            if isinstance(mask, np.ndarray) and mask.dtype == np.uint32:
                mask = mask.view(np.int32)
            mask = torch.as_tensor(mask)
            if mask.dtype == torch.uint32:
                mask = mask.view(torch.int32)
            if mask.dtype != torch.int32 or mask.dim() not in (1, 2):
                raise SamplerError("masks must be int32 or uint32 words [n, W]")
            self._take("mask", mask.unsqueeze(0) if mask.dim() == 1 else mask)
        if mask_of is not None:
            if mask is None:
                raise SamplerError("mask_of needs masks")
            self._take("mask_of", mask_of)
        if bias is not None:
            if all(d is None or isinstance(d, Mapping) for d in bias):
                bias = self._csr(bias)
            if len(bias) != 3:
                raise SamplerError("biases are one {token: bias} per record or CSR lists (ids, values, offsets)")
            ids, val, off = bias
            if not any(isinstance(t, torch.Tensor) and t.is_cuda for t in bias):
                self._check(np.asarray(ids, np.int64), np.asarray(val), np.asarray(off, np.int64))
            self._take("bias_ids", ids)
            self._take("bias", val)
            self._take("bias_off", off)
            if self.bias_ids.numel() != self.bias.numel() or self.bias_off.numel() < 1:
                raise SamplerError("biases are CSR lists (ids, values, offsets)")
        self.c = self._struct(self._held())

    def _as(self, name, x):
        """The array or tensor as the kernels read it."""
        if name != "mask":
            return _dev(x, {"bias": torch.float32, "bias_off": torch.int64}.get(name, torch.int32), self.device)
        x = x.to(self.device)
        packed = x.shape[1] <= 1 or x.stride(1) == 1
        return x if packed and (x.shape[0] <= 1 or x.stride(0) >= x.shape[1]) else x.contiguous()

    def _take(self, name, x):
        t = self._as(name, x)
        setattr(self, name, t)
        if isinstance(x, torch.Tensor) and x.device.type == self.device.type and t.data_ptr() != x.data_ptr():
            self._given[name] = x

    def _held(self):
        return {n: getattr(self, n) for n in ("mask", "mask_of", "bias_ids", "bias", "bias_off")
                if getattr(self, n) is not None}

    def _struct(self, held):
        """The fs_edits of device tensors, which it keeps."""
        c = FsEdits()
        c.tensors = list(held.values())

        def ptr(t):                                           # (no masks, no bias at all: a valid pointer, never read)
            if t.numel() == 0:
                t = torch.zeros(1, dtype=t.dtype, device=t.device)
                c.tensors.append(t)
            return t.data_ptr()

        mask, off = held.get("mask"), held.get("bias_off")
        if mask is not None:
            c.d_mask = ptr(mask)
            c.mask_ld = mask.stride(0) if mask.shape[0] > 1 else mask.shape[1]
            c.n_masks = mask.shape[0]
            c.d_mask_of = held["mask_of"].data_ptr() if "mask_of" in held else None
        if off is not None:
            c.d_bias_ids, c.d_bias, c.d_bias_off = ptr(held["bias_ids"]), ptr(held["bias"]), off.data_ptr()
        return c

    @staticmethod
    def _csr(dicts):
        rows = [sorted((int(t), float(b)) for t, b in (d or {}).items()) for d in dicts]
        off = np.zeros(len(rows) + 1, np.int64)
        off[1:] = np.cumsum([len(r) for r in rows])
        flat = [e for r in rows for e in r]
        return (np.array([t for t, _ in flat], np.int32), np.array([b for _, b in flat], np.float32), off)

    @staticmethod
    def _check(ids, val, off):
        if ids.ndim != 1 or val.shape != ids.shape or off.ndim != 1 or off.size < 1 or off[0] < 0 or off[-1] > ids.size \
                or np.any(np.diff(off) < 0):
            raise SamplerError("biases are CSR lists (ids, values, offsets)")
        step = np.diff(ids) < 0                               # descents are only allowed where a record begins
        step[[o - 1 for o in off if 0 < o < ids.size]] = False
        if np.any(step[off[0]:max(off[-1] - 1, off[0])]):
            raise SamplerError("the ids of a record's biases must ascend")

    @staticmethod
    def pack(allowed):
        """Mask words from truth values [n, V] (or [V]): int32 [n, ceil(V / 32)]."""
        if isinstance(allowed, torch.Tensor):
            a = allowed.bool()
            a = a.unsqueeze(0) if a.dim() == 1 else a
            a = torch.nn.functional.pad(a, (0, (-a.shape[1]) % 32)).view(a.shape[0], -1, 32)
            bit = 1 << torch.arange(32, dtype=torch.int64, device=a.device)
            return (a * bit).sum(2).to(torch.int32)
        a = np.atleast_2d(np.asarray(allowed, bool))
        a = np.pad(a, ((0, 0), (0, (-a.shape[1]) % 32)))
        return np.packbits(a, axis=1, bitorder="little").view(np.int32)

    def tensors(self):
        """The device tensors of the masks and biases."""
        return list(self._held().values())

    def _now(self, rows: int, records: int, V: int, dev):
        """The checked fs_edits for a call of `rows` logits rows and `records` records, on the current stream."""
        if dev != self.device:
            raise SamplerError(f"edits on {self.device}, logits on {dev}")
        if self.mask is not None:
            if self.mask.shape[1] * 32 < V:
                raise SamplerError(f"masks of {self.mask.shape[1]} words for {V} tokens")
            if (self.mask_of.numel() != rows) if self.mask_of is not None else (self.mask.shape[0] < rows):
                raise SamplerError("one mask index per row" if self.mask_of is not None else "one mask per row")
        if self.bias_off is not None and self.bias_off.numel() != records + 1:
            raise SamplerError("one bias list per record")
        if not self._given:
            return self.c
        return self._struct(dict(self._held(), **{n: self._as(n, x) for n, x in self._given.items()}))

    def _ref(self, rows: int, records: int, V: int, dev):
        return ctypes.byref(self._now(rows, records, V, dev))


def _on(stream, dev, *tensors):
    """The stream of a call on device `dev`, as the C ABI takes it. A stream other than the current one first waits for
    the current one, on which the wrapper's tensors are made, and is known to their allocator as a user."""
    cur = torch.cuda.current_stream(dev)
    if stream is not None and stream.cuda_stream != cur.cuda_stream:
        stream.wait_stream(cur)
        for t in tensors:
            if t is not None and t.is_cuda:
                t.record_stream(stream)
        return ctypes.c_void_p(stream.cuda_stream)
    return ctypes.c_void_p(cur.cuda_stream)


def sample_batch(logits, params, u, hist=None, hist_off=None, V=None, kcap=0, ctx=None, stream=None, route=None,
                 edits=None):
    """fs_sample_batch(_hp) on device tensors: logits [B, ld] fp32 (rows 16-byte aligned), params (B records),
    u [B] float64 draws, hist/hist_off CSR histories. Returns dict(tok, keep, cand_ids, cand_probs) (device).
    route: "host" / "device" (default: the module's ROUTE); params given as a device tensor always go "device".
    edits: an Edits, the masks and biases the rows are sampled under (fs_sample_edited); a row without a candidate has
    token -1."""
    logits, ld, n = _check_logits(logits, V)
    B = logits.shape[0]
    dev = logits.device
    p = _dev_params(params, dev)
    if p.numel() != B * PARAMS_DTYPE.itemsize:
        raise SamplerError("one params record per row")
    u = _dev(u, torch.float64, dev)
    if u.numel() < B:
        raise SamplerError("one draw per row")
    hist, hist_off = _hist_tensors(hist, hist_off, B, dev)
    tok = torch.empty(B, dtype=torch.int32, device=dev)
    keep = torch.empty(B, dtype=torch.int32, device=dev)
    ids = torch.empty((B, kcap), dtype=torch.int32, device=dev) if kcap else None
    probs = torch.empty((B, kcap), dtype=torch.float64, device=dev) if kcap else None
    ctx = ctx or Context.default(dev)
    hp = None                                             # the host copy of the parameters picks the kernel
    if (route or ROUTE) == "host" and not isinstance(params, torch.Tensor):
        hp = params_array(params)
    if edits is not None:
        with torch.cuda.device(dev), ctx.lock:
            ed = edits._now(B, B, n, dev)
            check(lib().fs_sample_edited(ctx.h, _lptr(logits), ld, B, n, _ptr(hist), _ptr(hist_off), _ptr(p), _hptr(hp),
                                         ctypes.byref(ed), _ptr(u), _ptr(tok), kcap, _ptr(ids), _ptr(probs), _ptr(keep),
                                         _on(stream, dev, logits, p, u, hist, hist_off, tok, keep, ids, probs,
                                             *ed.tensors)),
                  "fs_sample_edited")
        return dict(tok=tok, keep=keep, cand_ids=ids, cand_probs=probs, _keepalive=(p, u, hist, hist_off))
    with ctx.lock:
        if hp is not None:
            check(lib().fs_sample_batch_hp(ctx.h, _lptr(logits), ld, B, n, _ptr(hist), _ptr(hist_off), _ptr(p),
                                           hp.ctypes.data_as(ctypes.c_void_p), _ptr(u), _ptr(tok), kcap, _ptr(ids),
                                           _ptr(probs), _ptr(keep), _stream(stream)), "fs_sample_batch_hp")
        else:
            check(lib().fs_sample_batch(ctx.h, _lptr(logits), ld, B, n, _ptr(hist), _ptr(hist_off), _ptr(p),
                                        _ptr(u), _ptr(tok), kcap, _ptr(ids), _ptr(probs), _ptr(keep),
                                        _stream(stream)), "fs_sample_batch")
    return dict(tok=tok, keep=keep, cand_ids=ids, cand_probs=probs, _keepalive=(p, u, hist, hist_off))


def argmax_batch(logits, hist=None, hist_off=None, params=None, V=None, ctx=None, stream=None, edits=None):
    """fs_argmax_batch: greedy token per row after the penalties of `params` (None = no penalty). edits: the masks and
    biases of the rows (fs_sample_edited with greedy records); a row without a candidate has token -1."""
    if edits is not None:
        B = logits.shape[0] if logits.dim() == 2 else 1
        if isinstance(params, torch.Tensor):
            params = params.clone()
            params.view(torch.float32).view(-1, PARAMS_DTYPE.itemsize // 4)[:, 0] = 0.0
        else:
            g = np.zeros(B, PARAMS_DTYPE) if params is None else params_array(params).copy()
            g["temperature"] = 0.0
            if params is None:
                g["repetition_penalty"], g["top_p"], hist = 1.0, 1.0, None
            params = g
        return sample_batch(logits, params, np.zeros(B), hist=hist, hist_off=hist_off, V=V, ctx=ctx, stream=stream,
                            edits=edits)["tok"]
    logits, ld, n = _check_logits(logits, V)
    B = logits.shape[0]
    dev = logits.device
    p = _dev_params(params, dev) if params is not None else None
    hist, hist_off = _hist_tensors(hist, hist_off, B, dev)
    tok = torch.empty(B, dtype=torch.int32, device=dev)
    ctx = ctx or Context.default(dev)
    with ctx.lock:
        check(lib().fs_argmax_batch(ctx.h, _lptr(logits), ld, B, n, _ptr(hist), _ptr(hist_off), _ptr(p), _ptr(tok),
                                    _stream(stream)), "fs_argmax_batch")
    return tok


def verify(logits, rows, row_off, params, u=None, hist=None, hist_off=None, eos_id=-1, V=None, ctx=None,
           stream=None, route=None, edits=None):
    """fs_verify(_hp): per-row tokens and per-stream accepted prefix lengths of a speculative window. route as for
    sample_batch ("host": the host copy of the stream parameters goes along, fs_verify_hp). edits: masks by row and
    biases by stream (fs_verify_edited); a row without a candidate has token -1 and ends its window."""
    logits, ld, n = _check_logits(logits, V)
    R = logits.shape[0]
    dev = logits.device
    if not (isinstance(row_off, torch.Tensor) and row_off.is_cuda):
        o = np.asarray(row_off, np.int64)                 # (a row outside the windows would be counted as one of theirs)
        if o.ndim != 1 or o.size < 1 or o[0] != 0 or o[-1] != R or np.any(np.diff(o) < 0):
            raise SamplerError("row_off must ascend from 0 to the logits' rows")
    rows = _dev(rows, torch.int32, dev)
    row_off = _dev(row_off, torch.int64, dev)
    S = row_off.numel() - 1
    p = _dev_params(params, dev)
    if p.numel() != S * PARAMS_DTYPE.itemsize:
        raise SamplerError("one params record per stream")
    u = _dev(np.zeros(R) if u is None else u, torch.float64, dev)
    if rows.numel() < R or u.numel() < R:
        raise SamplerError("one fed token and one draw per row")
    hist, hist_off = _hist_tensors(hist, hist_off, S, dev)
    tok = torch.empty(R, dtype=torch.int32, device=dev)
    acc = torch.empty(S, dtype=torch.int32, device=dev)
    ctx = ctx or Context.default(dev)
    hp = None
    if (route or ROUTE) == "host" and not isinstance(params, torch.Tensor):
        hp = params_array(params)
    if edits is not None:
        with torch.cuda.device(dev), ctx.lock:
            ed = edits._now(R, S, n, dev)
            check(lib().fs_verify_edited(ctx.h, _lptr(logits), ld, S, R, n, _ptr(rows), _ptr(row_off), _ptr(hist),
                                         _ptr(hist_off), _ptr(p), _hptr(hp), ctypes.byref(ed), _ptr(u), int(eos_id),
                                         _ptr(tok), _ptr(acc),
                                         _on(stream, dev, logits, rows, row_off, p, u, hist, hist_off, tok, acc,
                                             *ed.tensors)),
                  "fs_verify_edited")
        return tok, acc
    with ctx.lock:
        if hp is not None:
            check(lib().fs_verify_hp(ctx.h, _lptr(logits), ld, S, R, n, _ptr(rows), _ptr(row_off), _ptr(hist),
                                     _ptr(hist_off), _ptr(p), hp.ctypes.data_as(ctypes.c_void_p), _ptr(u),
                                     int(eos_id), _ptr(tok), _ptr(acc), _stream(stream)), "fs_verify_hp")
        else:
            check(lib().fs_verify(ctx.h, _lptr(logits), ld, S, R, n, _ptr(rows), _ptr(row_off), _ptr(hist),
                                  _ptr(hist_off), _ptr(p), _ptr(u), int(eos_id), _ptr(tok), _ptr(acc),
                                  _stream(stream)), "fs_verify")
    return tok, acc


def penalize_batch(logits, params, hist=None, hist_off=None, V=None, ctx=None, stream=None):
    """fs_penalize_batch: leave each row penalised in place, as ferro's sample() leaves its host row
    (sampler.cpp:11-18). logits must be a writable [B, ld] fp32 CUDA tensor; returns it."""
    target = logits
    logits, ld, n = _check_logits(logits, V)
    B = logits.shape[0]
    dev = logits.device
    p = _dev_params(params, dev)
    if p.numel() != B * PARAMS_DTYPE.itemsize:
        raise SamplerError("one params record per row")
    hist, hist_off = _hist_tensors(hist, hist_off, B, dev)
    ctx = ctx or Context.default(dev)
    with ctx.lock:
        check(lib().fs_penalize_batch(ctx.h, _lptr(logits), ld, B, n, _ptr(hist), _ptr(hist_off), _ptr(p),
                                      _stream(stream)), "fs_penalize_batch")
    t2 = target if target.dim() == 2 else target.unsqueeze(0)
    if logits.data_ptr() != t2.data_ptr():            # repacked into an aligned copy: write the rows back
        t2[:, :n].copy_(logits[:, :n])
    return target


def lookup_draft(hist, hist_off, kmax, min_n=None, eos_id=-1, draft_ld=None, ctx=None, stream=None):
    """fs_lookup_draft: prompt-lookup drafts per stream (server.cpp:552-564). Returns (draft [S, draft_ld], n [S])."""
    hist_off = _dev(hist_off, torch.int64, "cuda")
    S = hist_off.numel() - 1
    dev = hist_off.device
    hist = _dev(hist, torch.int32, dev)
    km = _dev(np.broadcast_to(np.asarray(kmax, np.int32), (S,)).copy(), torch.int32, dev)
    mn = None if min_n is None else _dev(np.broadcast_to(np.asarray(min_n, np.int32), (S,)).copy(), torch.int32, dev)
    ld = int(draft_ld if draft_ld is not None else max(int(km.max().item()) if S else 1, 1))
    draft = torch.zeros((S, ld), dtype=torch.int32, device=dev)
    nd = torch.zeros(S, dtype=torch.int32, device=dev)
    ctx = ctx or Context.default(dev)
    with ctx.lock:
        check(lib().fs_lookup_draft(ctx.h, S, _ptr(hist), _ptr(hist_off), _ptr(km), _ptr(mn), int(eos_id),
                                    _ptr(draft), ld, _ptr(nd), _stream(stream)), "fs_lookup_draft")
    return draft, nd


def hist_append(hist, hist_off, tok, row_off=None, count=None, out_cap=None, ctx=None, stream=None):
    """fs_hist_append: each stream's consumed tokens pushed onto its history (server.cpp:342), on device CSR
    histories, out of place. Stream s gains tok[row_off[s] : row_off[s] + count[s]] (row_off None: row s; count
    None: 1 per stream; fs_verify's tok / row_off / accepted fit as they are). Returns (out_hist, out_off): out_off
    [S+1] int64 rebased to 0; out_hist holds out_cap ids (default: room for every row of tok), of which
    out_off[-1] are used. Stays on the device: nothing here waits for the GPU."""
    hist_off = _dev(hist_off, torch.int64, "cuda")
    dev = hist_off.device
    S = hist_off.numel() - 1
    hist = _dev(hist, torch.int32, dev)
    if hist.numel() == 0:
        hist = torch.zeros(1, dtype=torch.int32, device=dev)     # every history empty: a valid pointer, never read
    tok = _dev(tok, torch.int32, dev)
    ro = None if row_off is None else _dev(row_off, torch.int64, dev)
    cnt = None if count is None else _dev(count, torch.int32, dev)
    if ro is not None and ro.numel() != S + 1:
        raise SamplerError(f"row_off has {ro.numel()} entries for {S} streams")
    if cnt is not None and cnt.numel() != S:
        raise SamplerError(f"count has {cnt.numel()} entries for {S} streams")
    if out_cap is None:
        out_cap = hist.numel() + tok.numel()
    out = torch.empty(max(int(out_cap), 1), dtype=torch.int32, device=dev)
    out_off = torch.empty(S + 1, dtype=torch.int64, device=dev)
    ctx = ctx or Context.default(dev)
    with ctx.lock:
        check(lib().fs_hist_append(ctx.h, S, _ptr(hist), _ptr(hist_off), _ptr(tok), _ptr(ro), _ptr(cnt), _ptr(out),
                                   int(out_cap), _ptr(out_off), _stream(stream)), "fs_hist_append")
    return out, out_off


def decode_step(logits, params, rng, hist=None, hist_off=None, out_cap=None, V=None, ctx=None, stream=None,
                route=None, edits=None):
    """fs_decode_step(_hp): one decode step in one launch - each row's draw from its DeviceRng stream (row s = stream
    s), fs_sample_batch's token, and the token appended to the stream's history (server.cpp:603-606, then :342).
    Returns (tok, keep, out_hist, out_off); out_hist holds out_cap ids (default: room for one more per stream), of
    which out_off[-1] are used. Stays on the device. route as for sample_batch ("host": the host copy of the
    parameters goes along, fs_decode_step_hp). edits: the rows' masks and biases (fs_decode_step_edited); a row without a
    candidate appends token -1."""
    logits, ld, n = _check_logits(logits, V)
    B = logits.shape[0]
    dev = logits.device
    p = _dev_params(params, dev)
    if p.numel() != B * PARAMS_DTYPE.itemsize:
        raise SamplerError("one params record per row")
    if B > rng.n:
        raise SamplerError(f"{B} rows for {rng.n} draw streams")
    hist, hist_off = _hist_tensors(hist, hist_off, B, dev)
    if out_cap is None:
        out_cap = (hist.numel() if hist is not None else 0) + B
    tok = torch.empty(B, dtype=torch.int32, device=dev)
    keep = torch.empty(B, dtype=torch.int32, device=dev)
    out = torch.empty(max(int(out_cap), 1), dtype=torch.int32, device=dev)
    out_off = torch.empty(B + 1, dtype=torch.int64, device=dev)
    ctx = ctx or Context.default(dev)
    hp = params_array(params) if (route or ROUTE) == "host" and not isinstance(params, torch.Tensor) else None
    if edits is not None:
        with torch.cuda.device(dev), ctx.lock:
            ed = edits._now(B, B, n, dev)
            check(lib().fs_decode_step_edited(ctx.h, rng.h, _lptr(logits), ld, B, n, _ptr(hist), _ptr(hist_off), _ptr(p),
                                              _hptr(hp), ctypes.byref(ed), _ptr(tok), _ptr(keep), _ptr(out),
                                              _ptr(out_off), int(out_cap),
                                              _on(stream, dev, logits, p, hist, hist_off, tok, keep, out, out_off,
                                                  *ed.tensors)),
                  "fs_decode_step_edited")
        return tok, keep, out, out_off
    with ctx.lock:
        if hp is not None:
            check(lib().fs_decode_step_hp(ctx.h, rng.h, _lptr(logits), ld, B, n, _ptr(hist), _ptr(hist_off), _ptr(p),
                                          hp.ctypes.data_as(ctypes.c_void_p), _ptr(tok), _ptr(keep), _ptr(out),
                                          _ptr(out_off), int(out_cap), _stream(stream)), "fs_decode_step_hp")
        else:
            check(lib().fs_decode_step(ctx.h, rng.h, _lptr(logits), ld, B, n, _ptr(hist), _ptr(hist_off), _ptr(p),
                                       _ptr(tok), _ptr(keep), _ptr(out), _ptr(out_off), int(out_cap),
                                       _stream(stream)), "fs_decode_step")
    return tok, keep, out, out_off


_TYPES = {torch.float32: FS_F32, torch.bfloat16: FS_BF16, torch.float16: FS_F16}


def _typed_logits(logits, V):
    """(logits, ld, V, type) of a [B, ld] or [ld] device tensor of any type; other layouts are repacked."""
    if not (isinstance(logits, torch.Tensor) and logits.is_cuda and logits.dtype in _TYPES):
        raise SamplerError("logits must be a float32, bfloat16 or float16 CUDA tensor")
    if logits.dim() == 1:
        logits = logits.unsqueeze(0)
    if logits.dim() != 2:
        raise SamplerError("logits must be [B, V]")
    n = logits.shape[1] if V is None else V
    if n > logits.shape[1]:
        raise SamplerError("V exceeds the row length")
    ld = logits.stride(0) if logits.shape[0] > 1 else n + (-n) % 4
    if (n > 1 and logits.stride(1) != 1) or ld % 4 or ld < n or logits.data_ptr() % (4 * logits.element_size()) \
            or (logits.shape[0] == 1 and n % 4):              # (a lone row's last four must lie inside its buffer)
        padded = torch.zeros((logits.shape[0], n + (-n) % 4), dtype=logits.dtype, device=logits.device)
        padded[:, :n] = logits[:, :n]
        logits, ld = padded, padded.stride(0)
    return logits, ld, n, _TYPES[logits.dtype]


def edit_batch(logits, params=None, hist=None, hist_off=None, edits=None, V=None, out=None, ctx=None, stream=None):
    """fs_edit_batch: the edited logits in float32 [B, V] - softcap, biases, penalties, -inf where the row's mask does not
    allow a token. logits [B, ld] float32, bfloat16 or float16; params (B records; None: no softcap, no penalties).
    out: a float32 [B, >= V] tensor with 16-byte aligned rows, logits itself included (default: a new one); returned."""
    logits, ld, n, kind = _typed_logits(logits, V)
    B, dev = logits.shape[0], logits.device
    p = None
    if params is not None:
        p = _dev_params(params, dev)
        if p.numel() != B * PARAMS_DTYPE.itemsize:
            raise SamplerError("one params record per row")
    hist, hist_off = _hist_tensors(hist, hist_off, B, dev)
    if out is None:
        out = torch.empty((B, n + (-n) % 4), dtype=torch.float32, device=dev)[:, :n]
    o2 = out.unsqueeze(0) if out.dim() == 1 else out
    out_ld = o2.stride(0) if B > 1 else n + (-n) % 4
    if o2.dtype != torch.float32 or o2.device != dev or o2.dim() != 2 or o2.shape[0] != B or o2.shape[1] < n \
            or (o2.shape[1] > 1 and o2.stride(1) != 1):
        raise SamplerError("out must be a float32 [B, V] tensor on the logits' device with packed rows")
    if B == 1 and o2.data_ptr() == logits.data_ptr():
        out_ld = ld
    ctx = ctx or Context.default(dev)
    with torch.cuda.device(dev), ctx.lock:
        ed = None if edits is None else edits._now(B, B, n, dev)
        check(lib().fs_edit_batch(ctx.h, _lptr(logits), kind, ld, B, n, _ptr(hist), _ptr(hist_off), _ptr(p),
                                  None if ed is None else ctypes.byref(ed), ctypes.c_void_p(o2.data_ptr()), out_ld,
                                  _on(stream, dev, logits, p, hist, hist_off, out, *(ed.tensors if ed is not None else []))),
              "fs_edit_batch")
    return out


def logprobs(logits, tok=None, n=0, params=None, edits=None, V=None, ctx=None, stream=None):
    """fs_logprobs: log-probabilities under softmax((softcap(l) + bias) / T) over the allowed tokens. logits [B, ld]
    float32, bfloat16 or float16; params (B records, their softcap and temperature; None: the logits' own distribution).
    Returns dict(lp [B], rank [B]) of the tokens `tok` [B] and dict entries ids, top [B, n] of the n largest (None where
    not asked for)."""
    logits, ld, v, kind = _typed_logits(logits, V)
    B, dev = logits.shape[0], logits.device
    if not 0 <= n <= FS_MAX_TOP:
        raise SamplerError(f"n must lie in [0, {FS_MAX_TOP}]")
    p = None
    if params is not None:
        p = _dev_params(params, dev)
        if p.numel() != B * PARAMS_DTYPE.itemsize:
            raise SamplerError("one params record per row")
    t = lp = rank = ids = top = None
    if tok is not None:
        t = _dev(tok, torch.int32, dev)
        if t.numel() != B:
            raise SamplerError("one token per row")
        lp = torch.empty(B, dtype=torch.float32, device=dev)
        rank = torch.empty(B, dtype=torch.int32, device=dev)
    if n:
        ids = torch.empty((B, n), dtype=torch.int32, device=dev)
        top = torch.empty((B, n), dtype=torch.float32, device=dev)
    ctx = ctx or Context.default(dev)
    with torch.cuda.device(dev), ctx.lock:
        ed = None if edits is None else edits._now(B, B, v, dev)
        check(lib().fs_logprobs(ctx.h, _lptr(logits), kind, ld, B, v, _ptr(p), None if ed is None else ctypes.byref(ed),
                                _ptr(t), n, _ptr(lp), _ptr(rank), _ptr(ids), _ptr(top),
                                _on(stream, dev, logits, p, t, lp, rank, ids, top, *(ed.tensors if ed is not None else []))),
              "fs_logprobs")
    return dict(lp=lp, rank=rank, ids=ids, top=top)


def device_error(ctx=None, stream=None) -> int:
    ctx = ctx or Context.default()
    bits = ctypes.c_int32(0)
    check(lib().fs_device_error(ctx.h, _stream(stream), ctypes.byref(bits)), "fs_device_error")
    return bits.value


class Sampler:
    """Mirror of ferro::Sampler (src/sampler.h:23-34) running on the GPU.

    sample(logits, n_vocab, history) -> int, with logits a CUDA float32 tensor (device-resident, the intended
    use), a CPU tensor or a numpy float32 array (copied to the device). As in ferro (sampler.cpp:11-18) the row is
    left penalised in place, on whichever side it lives, unless the sampler was made with write_back=False (the
    token is the same either way: the kernels penalise on the fly)."""

    def __init__(self, p: SamplerParams, device=None, write_back: bool = True):
        self._p = p
        self._rng = Rng(int(p.seed))
        self._dev = torch.device("cuda" if device is None else device)
        self._rec = torch.from_numpy(params_array(p).view(np.uint8).copy()).to(self._dev)
        self._ctx = Context.default(self._dev)
        self._write_back = write_back

    def params(self) -> SamplerParams:
        return self._p

    def sample(self, logits, n_vocab: int, history) -> int:
        host = logits
        on_dev = isinstance(logits, torch.Tensor) and logits.is_cuda
        if not on_dev:
            logits = torch.as_tensor(np.asarray(logits, np.float32)).to(self._dev)
        row = logits.reshape(-1)[:n_vocab].reshape(1, -1)
        h = np.asarray(history, np.int32).reshape(-1)
        u = np.zeros(1) if self._p.is_greedy() else self._rng.next_u(1)
        hist_off = [0, h.size]
        out = sample_batch(row, self._rec, u, hist=h, hist_off=hist_off, V=n_vocab, ctx=self._ctx)
        tok = int(out["tok"].item())
        if self._write_back and h.size:
            penalize_batch(row, self._rec, hist=h, hist_off=hist_off, V=n_vocab, ctx=self._ctx)
            if not on_dev:
                pen = row.reshape(-1).cpu()
                if isinstance(host, torch.Tensor):
                    host.reshape(-1)[:n_vocab].copy_(pen)
                elif isinstance(host, np.ndarray) and host.dtype == np.float32:
                    host.reshape(-1)[:n_vocab] = pen.numpy()
        return tok
