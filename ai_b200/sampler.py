"""Device token sampler -- the reference's logits-in `_pick` (core/gengine.py:452-469) on one sm_100a kernel.

`pick(logits, temperature, top_p, rng, mask)` keeps the reference signature (rng: numpy Generator; it draws
exactly one `rng.random()` per sampled row, the same draw `Generator.choice(n, p)` makes, so a seeded rng
gives the reference's tokens). `sample(...)` adds top-k and repetition/presence/frequency penalties (no
reference counterpart; see aib_sample in include/ai_b200.h for the order of the steps). `adjust(...)` applies penalties,
biases and masks to a batch of requests that each have their own, before a draw.
"""
import numpy as np
import torch

from . import _lib
from ._lib import SampleParams, ptr, stream_ptr

PMAX = 4096


def params(temperature=0.0, top_k=0, top_p=1.0, repetition_penalty=1.0, presence_penalty=0.0,
           frequency_penalty=0.0):
    return SampleParams(float(temperature), int(top_k), float(top_p), float(repetition_penalty),
                        float(presence_penalty), float(frequency_penalty))


def workspace(B, V, device):
    """Scratch for the two-phase sampler path (slice partials + candidates); reuse it across calls."""
    n = _lib.lib().aib_sample_workspace(B, V)
    return torch.empty(max(n, 16), dtype=torch.uint8, device=device)


def sample_into(logits, out_ids, prm, u=None, prior=None, mask=None, B=None, ws=None):
    """Launch the sampler on rows [0, B) of logits [>=B, V] (fp32, CUDA) writing int64 ids into out_ids.
    u: float64 [B] CUDA tensor or None (greedy); prior: int32 [B, P] (-1 = empty); mask: int32 [B, ceil(V/32)];
    ws: uint8 workspace from `workspace(B, V)` (selects the multi-CTA path; None = one CTA per row)."""
    B = logits.shape[0] if B is None else B
    V = logits.shape[-1]
    ld = logits.stride(0) if logits.dim() > 1 else V
    n_prior = 0 if prior is None else prior.shape[-1]
    if prior is not None and prior.dtype != torch.int32:
        raise ValueError("prior ids must be int32")
    if mask is not None and (mask.dtype != torch.int32 or mask.shape[-1] != (V + 31) // 32):
        raise ValueError("mask must be int32 [B, ceil(V/32)]")
    _lib.call("aib_sample", ptr(logits), B, V, ld, prm, ptr(prior), n_prior, ptr(mask), ptr(u), ptr(out_ids),
              ptr(ws), 0 if ws is None else ws.numel(), stream_ptr())


def adjust(logits, out=None, prior=None, repetition=None, presence=None, frequency=None, bias_ids=None, bias=None,
           mask=None):
    """Penalties, biases and grammar masks of a batch of requests, each row with its own parameters (see
    aib_adjust_logits in include/ai_b200.h for the formula): logits [B, V] fp32 or bf16 CUDA rows -> out (default: in
    place; else it shares no memory with logits). repetition (> 0) / presence / frequency: fp32 [B] over the ids of prior (int32 [B, P], P <= 32767, -1 =
    empty); bias_ids int32 / bias fp32 [B, n], n <= 1024 (biases of an id listed twice add up, ids outside the
    vocabulary are ignored); mask int32 [B, ceil(V/32)], 1 = allowed. prior, biases and mask may be expanded from one
    row. Returns out."""
    if logits.dim() != 2 or logits.dtype not in (torch.float32, torch.bfloat16) or not logits.is_cuda:
        raise ValueError("adjust: logits must be fp32 or bf16 CUDA rows [B, V]")
    shape, dt, dev = logits.shape, logits.dtype, logits.device
    B, V = shape
    ld, step = logits.stride()
    at = out_at = logits.data_ptr()
    if out is None or out is logits:
        out, out_ld, out_step = logits, ld, step
    else:
        if out.shape != shape or out.dtype != dt or out.device != dev:
            raise ValueError("adjust: out must have the shape, type and device of logits")
        out_ld, out_step = out.stride()
        out_at = out.data_ptr()
    if (V > 1 and (step != 1 or out_step != 1)) or (B > 1 and out_ld < V):
        raise ValueError("adjust: rows must be contiguous and the rows of out apart")
    prior_at, prior_ld, n_prior = _side("prior", prior, B, torch.int32, dev)
    ids_at, ids_ld, nb = _side("bias_ids", bias_ids, B, torch.int32, dev)
    bias_at, bias_ld, nv = _side("bias", bias, B, torch.float32, dev)
    mask_at, mask_ld, words = _side("mask", mask, B, torch.int32, dev)
    if nb != nv:
        raise ValueError("adjust: bias_ids and bias go together")
    if mask is not None and words != (V + 31) // 32:
        raise ValueError("adjust: mask must have ceil(V/32) words a row")
    rep_at, pres_at, freq_at = (_per_row(n, t, B, dev) for n, t in (("repetition", repetition), ("presence", presence),
                                                                    ("frequency", frequency)))
    if B == 0 or V == 0:
        return out
    with _lib.on_device(dev.index) as stream:
        _lib.call("aib_adjust_logits", at, ld, out_at, out_ld, int(dt == torch.bfloat16), B, V, prior_at, prior_ld,
                  n_prior, rep_at, pres_at, freq_at, ids_at, ids_ld, bias_at, bias_ld, nb, mask_at, mask_ld, stream)
    return out


def _side(what, t, B, dtype, device):
    """Address, row stride and width of an optional [B, n] argument of `adjust`."""
    if t is None:
        return None, 0, 0
    shape, stride = t.shape, t.stride()
    if len(shape) != 2 or shape[0] != B or t.dtype != dtype or t.device != device or (shape[1] > 1 and stride[1] != 1):
        raise ValueError(f"adjust: {what} must be {dtype} [B, n] rows on the logits' device")
    return (t.data_ptr() if shape[1] else None), stride[0], shape[1]


def _per_row(what, t, B, device):
    if t is None:
        return None
    if t.dtype != torch.float32 or t.shape != (B,) or t.device != device or not t.is_contiguous():
        raise ValueError(f"adjust: {what} must be fp32 [B] on the logits' device")
    return t.data_ptr()


def sample(logits, temperature=0.0, top_p=1.0, top_k=0, us=None, prior=None, mask=None, repetition_penalty=1.0,
           presence_penalty=0.0, frequency_penalty=0.0, two_phase=True):
    """Convenience: returns a list of token ids. `us`: per-row uniform draws (sequence or tensor)."""
    if logits.dim() == 1:
        logits = logits[None]
    B = logits.shape[0]
    dev = logits.device
    out = torch.empty(B, dtype=torch.int64, device=dev)
    u = None
    if temperature > 0:
        if us is None:
            raise ValueError("sampling needs uniform draws")
        u = torch.as_tensor(np.asarray(us, np.float64)).to(dev)
    prm = params(temperature, top_k, top_p, repetition_penalty, presence_penalty, frequency_penalty)
    ws = workspace(B, logits.shape[-1], dev) if two_phase else None
    sample_into(logits.contiguous(), out, prm, u, prior, mask, ws=ws)
    return out.tolist()


def pick(logits, temperature=0.0, top_p=1.0, rng=None, mask=None):
    """GGUFEngine._pick semantics (gengine.py:452-469): logits [T, V]; mask = xgrammar-style int32 bitmask."""
    if logits.dim() == 1:
        logits = logits[None]
    us = None
    if temperature > 0:
        rng = rng or np.random.default_rng()
        us = [rng.random() for _ in range(logits.shape[0])]
    return sample(logits, temperature, top_p, 0, us, None, mask)
