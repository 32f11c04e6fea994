"""Autograd-visible operators over the C ABI (include/paccmann_hip.h).

torch is used for device memory, streams and the autograd graph only; every
arithmetic operation of the path runs in libpaccmann_hip.so.
"""
import ctypes
import math
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import check, load, ptr, require_device, stream_ptr


_PRECISIONS = {'fp32': 0, 'bf16': 1}


def set_matmul_precision(precision):
    """'fp32' (default; the mode parity with the reference is claimed on) or
    'bf16': the recurrent cells' products and the recurrent weight gradients
    take bf16-rounded operands with fp32 accumulation (pcm_set_matmul_precision).
    The reference trains in fp32 only (models/training.py:132-157)."""
    if precision not in _PRECISIONS:
        raise ValueError(
            f'precision {precision!r}: expected one of {sorted(_PRECISIONS)}'
        )
    check(
        load().pcm_set_matmul_precision(_PRECISIONS[precision]),
        'set_matmul_precision'
    )


def get_matmul_precision():
    mode = load().pcm_get_matmul_precision()
    return next(k for k, v in _PRECISIONS.items() if v == mode)


def _f32(t, what):
    require_device(t, what)
    if t.dtype != torch.float32:
        raise TypeError(f'{what}: expected float32, got {t.dtype}')
    return t


def _rows2d(x, what):
    """[.., K] tensor -> (tensor kept alive, rows, row stride) with unit
    column stride and a uniform row stride; copies only when it must."""
    k = x.shape[-1]
    x2 = x.reshape(-1, k)  # a view whenever the strides allow it
    if x2.stride(1) != 1 or (x2.shape[0] > 1 and x2.stride(0) < k):
        x2 = x2.contiguous()
    ld = x2.stride(0) if x2.shape[0] > 1 else max(k, 1)
    return x2, x2.shape[0], ld


def check_status(status, what='token ids'):
    """Raise the RuntimeError the reference's embedding lookup would raise for
    ids outside the vocabulary (generate_latent_codes.py:126 relies on it).
    One device->host read, so callers do it once per forward."""
    if status is None:
        return
    word = int(status.item())
    if word:
        status.zero_()
    if word & _lib.STATUS_TIMEOUT:
        raise _lib.PaccmannHipError(
            'the persistent forward kernel gave up waiting for its peer '
            'blocks (GPU shared with other work?); results are invalid -- '
            'set PCM_PERSIST=0 to use the launch chain'
        )
    if word & _lib.STATUS_BAD_TOKEN:
        raise RuntimeError(f'index out of range in self ({what})')
    if word & _lib.STATUS_BAD_PARENT:
        raise RuntimeError('index out of range in self (parents of beams)')


# Packed batches launch over the still-running prefix of the batch (True) or
# over every row, freezing the finished ones (False; also what happens when
# the lengths are not sorted).  Both give the same mu / logvar / loss /
# gradients; tests flip it to keep the frozen-row path covered.
SHRINK_ACTIVE_BATCH = True


def _active_rows(lengths, steps):
    """Host int32[T] of rows still running at each step, when the lengths
    (a CPU tensor, as pad_packed_sequence returns them) are sorted by
    decreasing length -- PackedSequence.batch_sizes, which the reference
    slices its hidden / stack by (utils/utils.py:226-243).  None otherwise:
    the kernels then run every row and freeze the finished ones."""
    if not SHRINK_ACTIVE_BATCH or lengths.device.type != 'cpu':
        return None
    lens = lengths.to(torch.int64)
    if lens.numel() == 0 or bool((lens[1:] > lens[:-1]).any()):
        return None
    steps_idx = torch.arange(steps).view(-1, 1)
    return (lens.view(1, -1) > steps_idx).sum(dim=1).to(torch.int32).contiguous()


def _direct_sinks(params, needs):
    """Gradient sinks (dp.GradSink) of ``params`` when EVERY wanted gradient
    can be written straight into its parameter's bucket view, all in the same
    state: (sinks, accumulate) with accumulate = 0 for the first write since
    ``zero_grad`` and 1 for a later one; None when any of them must take the
    ordinary route (a returned tensor that AccumulateGrad adds)."""
    sinks, states = [], set()
    for param, need in zip(params, needs):
        if param is None or not need:
            sinks.append(None)
            continue
        sink = getattr(param, '_pcm_grad_sink', None)
        if sink is None or not sink.usable_by(param):
            return None
        sinks.append(sink)
        states.add(sink.written)
    if len(states) != 1:
        return None
    return sinks, 1 if states.pop() else 0


def _host_ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


# --------------------------------------------------------------------------
# StackGRU over a sequence
# --------------------------------------------------------------------------
class StackGRUSequenceFn(torch.autograd.Function):
    """out[T,B,H], h_final[L,B,H], stack_final[B,D,W] =
    f(tokens[T,B], lengths, h0, stack0, *weights)."""

    @staticmethod
    def forward(ctx, cfg, tokens, lengths, h0, stack0, status, *weights):
        lib = load()
        require_device(tokens, 'StackGRU tokens')
        dims, n_layers = cfg['dims'], cfg['dims'].layers
        steps, batch = tokens.shape
        if batch != dims.batch:
            raise ValueError(f'batch {batch} != dims.batch {dims.batch}')
        dev = tokens.device
        tokens = tokens.contiguous()
        if tokens.dtype != torch.int64:
            tokens = tokens.long()
        training = 1 if cfg['training'] else 0
        hid = dims.hidden
        ctx.params = weights
        weights = [None if w is None else _f32(w, 'weight').contiguous()
                   for w in weights]
        wstruct = _lib.make_params(weights, n_layers)
        nbytes = lib.pcm_stackgru_saved_bytes(
            ctypes.byref(dims), steps, training
        )
        saved = torch.empty(nbytes // 4, dtype=torch.float32, device=dev)
        h_final = torch.empty(n_layers, batch, hid, device=dev)
        stack_final = None
        if dims.use_stack:
            stack_final = torch.empty(
                batch, dims.stack_depth, dims.stack_width, device=dev
            )
        h0_stride = 0
        if h0 is not None:
            _f32(h0, 'h0')
            if h0.dim() == 2:  # one [B,H] broadcast to every layer
                h0 = h0.contiguous()
                h0_stride = 0
            else:
                h0 = h0.contiguous()
                h0_stride = batch * hid
        if stack0 is not None:
            stack0 = _f32(stack0, 'stack0').contiguous()
        active = None
        if lengths is not None:
            active = _active_rows(lengths, steps)
            lengths = lengths.to(device=dev, dtype=torch.int32).contiguous()
        check(
            lib.pcm_stackgru_forward(
                ctypes.byref(dims), ctypes.byref(wstruct), ptr(tokens), steps,
                ptr(lengths), _host_ptr(active), ptr(h0), h0_stride,
                ptr(stack0),
                float(cfg['dropout']), int(cfg['seed']), training, ptr(saved),
                nbytes, ptr(h_final), ptr(stack_final), ptr(status),
                stream_ptr(dev)
            ), 'pcm_stackgru_forward'
        )
        off, ld = ctypes.c_size_t(), ctypes.c_size_t()
        check(
            lib.pcm_stackgru_out_view(
                ctypes.byref(dims), steps, training, ctypes.byref(off),
                ctypes.byref(ld)
            ), 'pcm_stackgru_out_view'
        )
        out = saved.as_strided(
            (steps, batch, hid), (batch * ld.value, ld.value, 1), off.value
        )
        ctx.cfg = cfg
        ctx.steps = steps
        ctx.h0_broadcast = h0 is not None and h0.dim() == 2
        ctx.has_h0 = h0 is not None
        ctx.has_stack0 = stack0 is not None
        ctx.saved_buf = saved
        ctx.tokens = tokens
        ctx.lengths = lengths
        ctx.active = active
        ctx.weights = weights
        ctx.set_materialize_grads(False)
        if stack_final is None:
            stack_final = torch.empty(0, device=dev)
            ctx.mark_non_differentiable(stack_final)
        return out, h_final, stack_final

    @staticmethod
    def backward(ctx, d_out, d_h_final, d_stack_final):
        lib = load()
        cfg = ctx.cfg
        if not cfg['training']:
            raise RuntimeError(
                'StackGRU backward needs a training-mode forward '
                '(module.train()): the eval-mode forward keeps no activations'
            )
        if ctx.saved_buf is None:
            raise RuntimeError(
                'StackGRU backward called twice: the saved activations are '
                'consumed by the first call (retain_graph is not supported)'
            )
        dims, n_layers = cfg['dims'], cfg['dims'].layers
        steps, batch, hid = ctx.steps, dims.batch, dims.hidden
        dev = ctx.tokens.device
        weights = ctx.weights
        wstruct = _lib.make_params(weights, n_layers)
        needs = ctx.needs_input_grad[6:]
        direct = _direct_sinks(ctx.params, needs)
        if direct is not None:
            sinks, accumulate = direct
            grads = [None if s is None else s.view for s in sinks]
        else:
            accumulate = 0
            grads = [
                torch.empty_like(w) if (w is not None and need) else None
                for w, need in zip(weights, needs)
            ]
        gstruct = _lib.make_params(grads, n_layers)
        d_out_ld = 0
        if d_out is not None:
            d_out = _f32(d_out, 'd_out')
            if d_out.stride(2) != 1 or d_out.stride(0) != batch * d_out.stride(1):
                d_out = d_out.contiguous()
            d_out_ld = d_out.stride(1)
        if d_h_final is not None:
            d_h_final = _f32(d_h_final, 'd_h_final').contiguous()
        if d_stack_final is not None and d_stack_final.numel() == 0:
            d_stack_final = None
        if d_stack_final is not None:
            d_stack_final = _f32(d_stack_final, 'd_stack_final').contiguous()
        d_h0 = None
        if ctx.has_h0 and ctx.needs_input_grad[3]:
            d_h0 = torch.empty(n_layers, batch, hid, device=dev)
        d_stack0 = None
        if ctx.has_stack0 and ctx.needs_input_grad[4] and dims.use_stack:
            d_stack0 = torch.empty(
                batch, dims.stack_depth, dims.stack_width, device=dev
            )
        sbytes = lib.pcm_stackgru_scratch_bytes(ctypes.byref(dims), steps)
        scratch = torch.empty(sbytes // 4, dtype=torch.float32, device=dev)
        saved = ctx.saved_buf
        check(
            lib.pcm_stackgru_backward(
                ctypes.byref(dims), ctypes.byref(wstruct), ptr(ctx.tokens),
                steps, ptr(ctx.lengths), _host_ptr(ctx.active),
                float(cfg['dropout']),
                int(cfg['seed']), ptr(saved), saved.numel() * 4, ptr(d_out),
                d_out_ld, ptr(d_h_final), ptr(d_stack_final), ptr(d_h0),
                ptr(d_stack0), ctypes.byref(gstruct), accumulate, ptr(scratch),
                sbytes, stream_ptr(dev)
            ), 'pcm_stackgru_backward'
        )
        ctx.saved_buf = None
        pad = cfg.get('pad_index')
        if grads[4] is not None and pad is not None:
            grads[4][pad].zero_()  # nn.Embedding(padding_idx=...) semantics
        if d_h0 is not None and ctx.h0_broadcast:
            d_h0 = d_h0.sum(dim=0)
        if direct is not None:
            # written in place: nothing for AccumulateGrad to add
            for sink in sinks:
                if sink is not None:
                    sink.mark_written()
            grads = [None] * len(grads)
        ctx.params = None
        return (None, None, None, d_h0, d_stack0, None) + tuple(grads)


# --------------------------------------------------------------------------
# dense layer
# --------------------------------------------------------------------------
_scratch_cache = {}


def _linear_scratch(dev, m, n, k):
    """One reusable scratch buffer per (device, stream): calls on a stream are
    ordered and the buffer is only used inside a single library call; two
    streams (two host threads, or the two directions of a bidirectional
    encoder) must not share one."""
    lib = load()
    need = lib.pcm_linear_scratch_bytes(m, n, k)
    key = (dev, torch.cuda.current_stream(dev).cuda_stream)
    buf = _scratch_cache.get(key)
    if buf is None or buf.numel() * 4 < need:
        if len(_scratch_cache) >= 16:   # streams come and go: do not hoard
            _scratch_cache.clear()
        buf = torch.empty(need // 4 + 1, dtype=torch.float32, device=dev)
        _scratch_cache[key] = buf
    return buf


class LinearFn(torch.autograd.Function):
    """y = x . w^T + b on the fp32 MFMA GEMM (torch.nn.Linear semantics)."""

    @staticmethod
    def forward(ctx, x, weight, bias):
        lib = load()
        _f32(x, 'linear input')
        weight_param, bias_param = weight, bias
        weight = _f32(weight, 'linear weight').contiguous()
        n, k = weight.shape
        x2, m, ldx = _rows2d(x, 'linear input')
        y = torch.empty(x.shape[:-1] + (n, ), device=x.device)
        if bias is not None:
            bias = _f32(bias, 'linear bias').contiguous()
        check(
            lib.pcm_linear_forward(
                ptr(x2), ldx, ptr(weight), ptr(bias), ptr(y), n, m, n, k,
                stream_ptr(x.device)
            ), 'pcm_linear_forward'
        )
        ctx.save_for_backward(x2, weight)
        ctx.ldx = ldx
        ctx.in_shape = x.shape
        ctx.has_bias = bias is not None
        ctx.params = (weight_param, bias_param)
        return y

    @staticmethod
    def backward(ctx, dy):
        lib = load()
        x2, weight = ctx.saved_tensors
        n, k = weight.shape
        dy2, m, lddy = _rows2d(_f32(dy, 'linear grad'), 'linear grad')
        dev = dy.device
        need_x, need_w, need_b = ctx.needs_input_grad
        dx = torch.empty(m, k, device=dev) if need_x else None
        need_b = need_b and ctx.has_bias
        direct = _direct_sinks(ctx.params, (need_w, need_b))
        accumulate = 0
        if direct is not None:
            (sink_w, sink_b), accumulate = direct
            dw = sink_w.view if sink_w is not None else None
            db = sink_b.view if sink_b is not None else None
        else:
            dw = torch.empty(n, k, device=dev) if need_w else None
            db = torch.empty(n, device=dev) if need_b else None
        scratch = _linear_scratch(dev, m, n, k)
        check(
            lib.pcm_linear_backward(
                ptr(x2), ctx.ldx, ptr(weight), ptr(dy2), None, lddy, ptr(dx),
                k, ptr(dw), ptr(db), m, n, k, accumulate, ptr(scratch),
                scratch.numel() * 4, stream_ptr(dev)
            ), 'pcm_linear_backward'
        )
        if dx is not None:
            dx = dx.view(ctx.in_shape)
        if direct is not None:
            for sink in (sink_w, sink_b):
                if sink is not None:
                    sink.mark_written()
            dw = db = None
        return dx, dw, db


def linear(x, weight, bias=None):
    return LinearFn.apply(x, weight, bias)


# --------------------------------------------------------------------------
# decoder head: logits + cross entropy summed over steps (vae.py:342-343)
# --------------------------------------------------------------------------
class DecoderHeadFn(torch.autograd.Function):
    """loss, argmax[B,T], logits[T,B,V] = head(out[T,B,H], W, b, targets)."""

    @staticmethod
    def forward(ctx, out, weight, bias, targets, lengths, status,
                step_weight=None):
        lib = load()
        _f32(out, 'decoder outputs')
        steps, batch, hid = out.shape
        ctx.params = (weight, bias)
        weight = _f32(weight, 'output_layer.weight').contiguous()
        bias = _f32(bias, 'output_layer.bias').contiguous()
        vocab = weight.shape[0]
        dev = out.device
        x2, m, ldx = _rows2d(out, 'decoder outputs')
        logits = torch.empty(steps, batch, vocab, device=dev)
        targets = targets.to(device=dev, dtype=torch.int64).contiguous()
        if lengths is not None:
            lengths = lengths.to(device=dev, dtype=torch.int32).contiguous()
        loss = torch.empty((), device=dev)
        argmax = torch.empty(batch, steps, dtype=torch.int64, device=dev)
        want_grad = any(ctx.needs_input_grad[:3])
        dlogits = torch.empty_like(logits) if want_grad else None
        scratch = torch.empty(m + steps, device=dev)
        if step_weight is not None:
            # data parallel: 1 / (rows active at step t over all ranks)
            step_weight = step_weight.to(
                device=dev, dtype=torch.float32
            ).contiguous()
            if step_weight.numel() != steps:
                raise ValueError('step_weight must have one entry per step')
        # output layer, softmax, cross entropy and argmax in one kernel
        check(
            lib.pcm_output_ce(
                ptr(x2), ldx, ptr(weight), ptr(bias), ptr(targets),
                ptr(lengths), ptr(step_weight), steps, batch, vocab, hid,
                ptr(logits), ptr(loss), ptr(argmax), ptr(dlogits),
                ptr(scratch), ptr(status), stream_ptr(dev)
            ), 'pcm_output_ce'
        )
        ctx.save_for_backward(x2, weight)
        ctx.dlogits = dlogits
        ctx.ldx = ldx
        ctx.shape = (steps, batch, hid, vocab)
        ctx.mark_non_differentiable(argmax, logits)
        return loss, argmax, logits

    @staticmethod
    def backward(ctx, dloss, _dargmax, _dlogits):
        lib = load()
        x2, weight = ctx.saved_tensors
        steps, batch, hid, vocab = ctx.shape
        m = steps * batch
        dev = x2.device
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dx = torch.empty(steps, batch, hid, device=dev) if need_x else None
        direct = _direct_sinks(ctx.params, (need_w, need_b))
        accumulate = 0
        if direct is not None:
            (sink_w, sink_b), accumulate = direct
            dw = sink_w.view if sink_w is not None else None
            db = sink_b.view if sink_b is not None else None
        else:
            dw = torch.empty(vocab, hid, device=dev) if need_w else None
            db = torch.empty(vocab, device=dev) if need_b else None
        dloss = _f32(dloss, 'dloss').reshape(1).contiguous()
        scratch = _linear_scratch(dev, m, vocab, hid)
        check(
            lib.pcm_linear_backward(
                ptr(x2), ctx.ldx, ptr(weight), ptr(ctx.dlogits), ptr(dloss),
                vocab, ptr(dx), hid, ptr(dw), ptr(db), m, vocab, hid,
                accumulate, ptr(scratch), scratch.numel() * 4, stream_ptr(dev)
            ), 'pcm_linear_backward(output_layer)'
        )
        ctx.dlogits = None
        if direct is not None:
            for sink in (sink_w, sink_b):
                if sink is not None:
                    sink.mark_written()
            dw = db = None
        return dx, dw, db, None, None, None, None


# --------------------------------------------------------------------------
# latent
# --------------------------------------------------------------------------
class ReparamFn(torch.autograd.Function):
    """z = eps * exp(0.5*logvar) + mu (vae.py:538-540)."""

    @staticmethod
    def forward(ctx, mu, logvar, eps):
        lib = load()
        mu = _f32(mu, 'mu').contiguous()
        logvar = _f32(logvar, 'logvar').contiguous()
        eps = _f32(eps, 'eps').contiguous()
        z = torch.empty_like(mu)
        check(
            lib.pcm_reparam_forward(
                ptr(mu), ptr(logvar), ptr(eps), ptr(z), mu.numel(),
                stream_ptr(mu.device)
            ), 'pcm_reparam_forward'
        )
        ctx.save_for_backward(logvar, eps)
        return z

    @staticmethod
    def backward(ctx, dz):
        lib = load()
        logvar, eps = ctx.saved_tensors
        dz = _f32(dz, 'dz').contiguous()
        dmu = torch.empty_like(dz) if ctx.needs_input_grad[0] else None
        dlv = torch.empty_like(dz) if ctx.needs_input_grad[1] else None
        check(
            lib.pcm_reparam_backward(
                ptr(dz), ptr(logvar), ptr(eps), ptr(dmu), ptr(dlv),
                dz.numel(), stream_ptr(dz.device)
            ), 'pcm_reparam_backward'
        )
        return dmu, dlv, None


class KLDivFn(torch.autograd.Function):
    """-0.5 * sum(1 + logvar - mu^2 - exp(logvar)) (loss_functions.py:39)."""

    @staticmethod
    def forward(ctx, mu, logvar):
        lib = load()
        mu = _f32(mu, 'mu').contiguous()
        logvar = _f32(logvar, 'logvar').contiguous()
        n = mu.numel()
        kl = torch.empty((), device=mu.device)
        scratch = torch.empty(
            max(1, lib.pcm_kl_scratch_floats(n)), device=mu.device
        )
        check(
            lib.pcm_kl_forward(
                ptr(mu), ptr(logvar), ptr(kl), ptr(scratch), n,
                stream_ptr(mu.device)
            ), 'pcm_kl_forward'
        )
        ctx.save_for_backward(mu, logvar)
        return kl

    @staticmethod
    def backward(ctx, dkl):
        lib = load()
        mu, logvar = ctx.saved_tensors
        dkl = _f32(dkl, 'dkl').reshape(1).contiguous()
        dmu = torch.empty_like(mu) if ctx.needs_input_grad[0] else None
        dlv = torch.empty_like(mu) if ctx.needs_input_grad[1] else None
        check(
            lib.pcm_kl_backward(
                ptr(dkl), ptr(mu), ptr(logvar), ptr(dmu), ptr(dlv),
                mu.numel(), stream_ptr(mu.device)
            ), 'pcm_kl_backward'
        )
        return dmu, dlv


# --------------------------------------------------------------------------
# generation (no autograd)
# --------------------------------------------------------------------------
def stackgru_generate(
    dims, weights, out_w, out_b, h0, prime, generate_len, search, temperature,
    seed, want_logits=False, status=None
):
    """pcm_stackgru_generate; h0 is [B,H] (broadcast) or [L,B,H].  Returns
    (tokens i64[B, P+G], logits [G,B,V] or None)."""
    lib = load()
    require_device(h0, 'generate h0')
    dev = h0.device
    n_layers, batch, hid = dims.layers, dims.batch, dims.hidden
    weights = [None if w is None else _f32(w, 'weight').contiguous()
               for w in weights]
    wstruct = _lib.make_params(weights, n_layers)
    h0 = _f32(h0, 'h0').contiguous()
    h0_stride = 0 if h0.dim() == 2 else batch * hid
    prime = prime.to(device=dev, dtype=torch.int64).contiguous().view(-1)
    plen = prime.numel()
    tokens = torch.empty(batch, plen + generate_len, dtype=torch.int64,
                         device=dev)
    logits = None
    if want_logits and generate_len > 0:
        logits = torch.empty(generate_len, batch, dims.vocab, device=dev)
    nbytes = lib.pcm_generate_workspace_bytes(ctypes.byref(dims))
    work = torch.empty(nbytes // 4, dtype=torch.float32, device=dev)
    out_w = _f32(out_w, 'output_layer.weight').contiguous()
    out_b = _f32(out_b, 'output_layer.bias').contiguous()
    check(
        lib.pcm_stackgru_generate(
            ctypes.byref(dims), ctypes.byref(wstruct), ptr(out_w), ptr(out_b),
            ptr(h0), h0_stride, ptr(prime), plen, int(generate_len),
            int(search), float(temperature), int(seed), ptr(tokens),
            ptr(logits), ptr(work), nbytes, ptr(status), stream_ptr(dev)
        ), 'pcm_stackgru_generate'
    )
    return tokens, logits


def stackgru_generate_beam(
    dims, weights, out_w, out_b, h0, prime, generate_len, beam_width,
    top_tokens, temperature, want_beams=False, status=None
):
    """pcm_stackgru_generate_beam; h0 is [B,H] (broadcast) or [L,B,H].
    Returns tokens i64[B, G] (the best beam of every row, without the prime),
    and with ``want_beams`` also (beam tokens i64[B, width, G], scores
    f64[B, width])."""
    lib = load()
    require_device(h0, 'generate h0')
    dev = h0.device
    n_layers, batch, hid = dims.layers, dims.batch, dims.hidden
    weights = [None if w is None else _f32(w, 'weight').contiguous()
               for w in weights]
    wstruct = _lib.make_params(weights, n_layers)
    h0 = _f32(h0, 'h0').contiguous()
    h0_stride = 0 if h0.dim() == 2 else batch * hid
    prime = prime.to(device=dev, dtype=torch.int64).contiguous().view(-1)
    tokens = torch.empty(batch, generate_len, dtype=torch.int64, device=dev)
    beams = scores = None
    if want_beams:
        beams = torch.empty(batch, beam_width, generate_len,
                            dtype=torch.int64, device=dev)
        scores = torch.empty(batch, beam_width, dtype=torch.float64,
                             device=dev)
    nbytes = lib.pcm_generate_beam_workspace_bytes(
        ctypes.byref(dims), int(beam_width), int(generate_len)
    )
    if nbytes == 0:
        check(-1, 'pcm_generate_beam_workspace_bytes')
    work = torch.empty(nbytes // 4, dtype=torch.float32, device=dev)
    out_w = _f32(out_w, 'output_layer.weight').contiguous()
    out_b = _f32(out_b, 'output_layer.bias').contiguous()
    check(
        lib.pcm_stackgru_generate_beam(
            ctypes.byref(dims), ctypes.byref(wstruct), ptr(out_w), ptr(out_b),
            ptr(h0), h0_stride, ptr(prime), prime.numel(), int(generate_len),
            int(beam_width), int(top_tokens), float(temperature), ptr(tokens),
            ptr(beams), ptr(scores), ptr(work), nbytes, ptr(status),
            stream_ptr(dev)
        ), 'pcm_stackgru_generate_beam'
    )
    if want_beams:
        return tokens, beams, scores
    return tokens


def search_step(logits, search, temperature=1.0, seed=0, step=0):
    """pcm_search_step: one token per row of ``logits[..., V]`` (a GPU
    tensor); returns i64 of shape ``logits.shape[:-1]``."""
    lib = load()
    require_device(logits, 'search logits')
    x2, rows, ld = _rows2d(_f32(logits, 'search logits'), 'search logits')
    if ld != x2.shape[1]:
        x2 = x2.contiguous()
    out = torch.empty(rows, dtype=torch.int64, device=logits.device)
    check(
        lib.pcm_search_step(
            ptr(x2), rows, x2.shape[1], int(search), float(temperature),
            int(seed), int(step), ptr(out), stream_ptr(logits.device)
        ), 'pcm_search_step'
    )
    return out.view(logits.shape[:-1])


def stackgru_generate_joint_beam(
    dims, weights, out_w, out_b, h0, prime, generate_len, beam_width,
    temperature, end_token=None, want_beams=False, status=None
):
    """pcm_stackgru_generate_joint_beam; h0 is [B,H] (broadcast) or [L,B,H],
    ``end_token`` None, a number or a tensor of one (on the device it is read
    there).  Returns tokens i64[B, G] (the best beam of every row, without the
    prime), and with ``want_beams`` also (beam tokens i64[B, width, G], scores
    f64[B, width]), best first."""
    lib = load()
    require_device(h0, 'generate h0')
    dev = h0.device
    n_layers, batch, hid = dims.layers, dims.batch, dims.hidden
    weights = [None if w is None else _f32(w, 'weight').contiguous()
               for w in weights]
    wstruct = _lib.make_params(weights, n_layers)
    h0 = _f32(h0, 'h0').contiguous()
    h0_stride = 0 if h0.dim() == 2 else batch * hid
    prime = prime.to(device=dev, dtype=torch.int64).contiguous().view(-1)
    tokens = torch.empty(batch, generate_len, dtype=torch.int64, device=dev)
    beams = scores = None
    if want_beams:
        beams = torch.empty(batch, beam_width, generate_len,
                            dtype=torch.int64, device=dev)
        scores = torch.empty(batch, beam_width, dtype=torch.float64,
                             device=dev)
    nbytes = lib.pcm_generate_joint_beam_workspace_bytes(
        ctypes.byref(dims), int(beam_width), int(generate_len)
    )
    if nbytes == 0:
        check(-1, 'pcm_generate_joint_beam_workspace_bytes')
    work = torch.empty(nbytes // 4, dtype=torch.float32, device=dev)
    out_w = _f32(out_w, 'output_layer.weight').contiguous()
    out_b = _f32(out_b, 'output_layer.bias').contiguous()
    call = lib.pcm_stackgru_generate_joint_beam
    if end_token is None:
        end = -1
    elif torch.is_tensor(end_token) and end_token.is_cuda:
        call = lib.pcm_stackgru_generate_joint_beam_until
        end_token = end_token.reshape(-1)[0].to(device=dev, dtype=torch.int64)
        end = end_token.data_ptr()
    else:
        end = int(torch.as_tensor(end_token).reshape(-1)[0])
    with _on(dev):
        check(
            call(
                ctypes.byref(dims), ctypes.byref(wstruct), ptr(out_w),
                ptr(out_b), ptr(h0), h0_stride, ptr(prime), prime.numel(),
                int(generate_len), int(beam_width), float(temperature),
                end, ptr(tokens), ptr(beams), ptr(scores), ptr(work), nbytes,
                ptr(status), stream_ptr(dev)
            ), 'pcm_stackgru_generate_joint_beam'
        )
    if want_beams:
        return tokens, beams, scores
    return tokens


# --------------------------------------------------------------------------
# top logits, distillation, joint beam search
#
# A serving loop or a small batch is bound by what a call costs on the host, so
# what is well-formed passes one comparison per tensor here and only the rest is
# looked at for what is wrong with it.
# --------------------------------------------------------------------------
class _Here:
    """A context that is nothing: the device is current already."""

    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return False


_HERE = _Here()


def _on(device):
    """Makes ``device`` the current one for a library call."""
    if torch.cuda.current_device() == device.index:
        return _HERE
    return torch.cuda.device(device)


def _stream(device):
    """``stream_ptr`` without the Python object around it (2 us)."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def _has_tangent(t):
    """Whether ``t`` carries a derivative in forward mode."""
    # (outside a dual level nothing does: the usual case costs 0.1 us)
    if getattr(forward_ad, '_current_level', 0) < 0 or t is None:
        return False
    return forward_ad.unpack_dual(t).tangent is not None


def _dtype_code(t, what):
    code = _lib.DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(
            f'{what}: expected float32, bfloat16 or float16, got {t.dtype}'
        )
    return code


def _operand(t, what, device, shape, *dtypes):
    """``t`` on ``device``, of that shape and one of those types, dense."""
    if t.device != device:
        raise ValueError(f'{what} is on {t.device}, the logits on {device}')
    if t.dtype not in dtypes:
        names = ' or '.join(str(d).split('.')[-1] for d in dtypes)
        raise TypeError(f'{what}: expected {names}, got {t.dtype}')
    if t.shape != shape:
        raise ValueError(
            f'{what} has shape {tuple(t.shape)}, expected {tuple(shape)}'
        )
    return t if t.is_contiguous() else t.contiguous()


def _status_word(status, device):
    if status is not None and (status.dtype != torch.int32
                               or status.device != device
                               or status.numel() != 1):
        raise ValueError(f'status: expected one int32 on {device}')
    return status


def _rows_of(x, what):
    """(tensor kept alive, rows, row stride) of ``x[..., V]``."""
    if x.is_contiguous():
        vocab = x.shape[-1]
        return x, x.numel() // vocab, vocab
    return _rows2d(x, what)


def _check_temperature(temperature):
    temperature = float(temperature)
    if not 1e-30 < temperature < 1e30:
        raise ValueError(f'temperature {temperature} must be positive')
    return temperature


def _check_vocab(vocab):
    if not 1 <= vocab <= _lib.MAX_VOCAB:
        raise ValueError(
            f'vocabulary of {vocab}: expected 1..{_lib.MAX_VOCAB}'
        )


class TopLogits(NamedTuple):
    """What ``top_logits`` keeps of a teacher and ``distill_loss`` takes:
    the largest logits (their own type) and their indices i32[..., k], the
    log-sum-exp f32[...] of the others at ``temperature`` (None: they are given
    no probability), and that temperature.  A negative index marks an entry
    that is absent, so that lists of different lengths fit one tensor."""
    values: torch.Tensor
    indices: torch.Tensor
    rest: Optional[torch.Tensor] = None
    temperature: float = 1.0


def top_logits(logits, k, temperature=1.0):
    """The ``k`` largest of ``logits[..., V]`` (fp32, bf16 or fp16), largest
    first, equal ones by index, with log sum exp(logits / temperature) over the
    others: ``TopLogits`` of shapes [..., k], [..., k], [...].  No gradient.  A
    NaN ranks below every number and makes its row's ``rest`` NaN."""
    lib = load()
    require_device(logits, 'top logits')
    code = _dtype_code(logits, 'top logits')
    temperature = _check_temperature(temperature)
    if logits.dim() < 1:
        raise ValueError('top logits: a row of logits is needed')
    vocab = logits.shape[-1]
    _check_vocab(vocab)
    k = int(k)
    if not 1 <= k <= min(vocab, _lib.TOP_MAX):
        raise ValueError(
            f'k={k}: expected 1..{min(vocab, _lib.TOP_MAX)} '
            f'(vocabulary {vocab})'
        )
    dev, lead = logits.device, logits.shape[:-1]
    listed = lead + (k, )
    values = torch.empty(listed, dtype=logits.dtype, device=dev)
    indices = torch.empty(listed, dtype=torch.int32, device=dev)
    rest = torch.empty(lead, dtype=torch.float32, device=dev)
    if rest.numel():
        x2, rows, ld = _rows_of(logits.detach(), 'top logits')
        need = lib.pcm_top_logits_workspace_bytes(rows, vocab, k)
        work = None
        if need:
            work = torch.empty(need, dtype=torch.uint8, device=dev)
        with _on(dev):
            check(
                lib.pcm_top_logits(
                    x2.data_ptr(), code, rows, ld, vocab, k, temperature,
                    values.data_ptr(), indices.data_ptr(), rest.data_ptr(),
                    ptr(work), need, _stream(dev)
                ), 'pcm_top_logits'
            )
    return TopLogits(values, indices, rest, temperature)


def _distill(logits, want, args):
    """pcm_distill_loss on checked operands: (loss, dlogits or None, scratch)."""
    (code, vocab, values, indices, rest, temperature, targets, lengths,
     hard_weight, step_weight, status) = args
    lib = load()
    steps, batch, _ = logits.shape
    dev = logits.device
    x2, _, ld = _rows_of(logits, 'distill logits')
    loss = torch.empty((), device=dev)
    dlogits = None
    if want:
        dlogits = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
    scratch = torch.empty(
        lib.pcm_distill_scratch_floats(steps, batch), device=dev
    )
    with _on(dev):
        check(
            lib.pcm_distill_loss(
                x2.data_ptr(), code, ld, values.data_ptr(),
                _lib.DTYPES[values.dtype], indices.data_ptr(), ptr(rest),
                indices.shape[-1], ptr(targets), ptr(lengths),
                ptr(step_weight), steps, batch, vocab, temperature,
                hard_weight, loss.data_ptr(), ptr(dlogits),
                scratch.data_ptr(), ptr(status), _stream(dev)
            ), 'pcm_distill_loss'
        )
    return loss, dlogits, scratch


def _refuse_create_graph():
    """In a ``backward``: the gradient would be a constant of that graph, and a
    second derivative through it silently lack this loss."""
    if torch.is_grad_enabled():
        raise RuntimeError(
            'distill_loss has no second derivative (backward with '
            'create_graph)'
        )


class DistillLossFn(torch.autograd.Function):
    """loss = distill(logits[T,B,V], teacher); the gradient is computed with
    the loss and multiplied by the incoming one in ``backward``."""

    @staticmethod
    def forward(ctx, logits, args):
        loss, dlogits, _ = _distill(logits, True, args)
        ctx.dlogits = dlogits
        ctx.scale = (dlogits.data_ptr(), args[0], dlogits.numel())
        return loss

    @staticmethod
    def backward(ctx, dloss):
        dlogits = ctx.dlogits
        if dlogits is None:
            raise RuntimeError(
                'distill_loss backward called twice: the gradient is handed '
                'out by the first call (retain_graph is not supported)'
            )
        _refuse_create_graph()
        ctx.dlogits = None
        # (an fp32 scalar; autograd's thread has the device and the stream of
        # the forward)
        check(
            load().pcm_scale(
                *ctx.scale, dloss.data_ptr(), _stream(dloss.device)
            ), 'pcm_scale'
        )
        return dlogits, None


class DistillHalfLossFn(torch.autograd.Function):
    """The same for fp16: the gradient is computed in ``backward``, where the
    incoming one goes in before the rounding (a loss scale keeps what fp16
    cannot hold without it).  The logits are read once more for it."""

    @staticmethod
    def forward(ctx, logits, args):
        (code, vocab, values, indices, rest, temperature, targets, lengths,
         hard_weight, step_weight, _) = args
        loss, _, scratch = _distill(logits, False, args)
        ctx.save_for_backward(logits, values, indices, rest, targets, lengths,
                              step_weight, scratch)
        ctx.scalars = code, vocab, temperature, hard_weight
        return loss

    @staticmethod
    def backward(ctx, dloss):
        _refuse_create_graph()
        (logits, values, indices, rest, targets, lengths, step_weight,
         scratch) = ctx.saved_tensors
        code, vocab, temperature, hard_weight = ctx.scalars
        steps, batch, _ = logits.shape
        dev = logits.device
        x2, _, ld = _rows_of(logits, 'distill logits')
        dlogits = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
        weights = ptr(step_weight)
        if weights is None and lengths is not None:   # the forward's
            weights = scratch.data_ptr() + 4 * steps * batch
        check(
            load().pcm_distill_grad(
                x2.data_ptr(), code, ld, values.data_ptr(),
                _lib.DTYPES[values.dtype], indices.data_ptr(), ptr(rest),
                indices.shape[-1], ptr(targets), ptr(lengths), weights, steps,
                batch, vocab, temperature, hard_weight, dloss.data_ptr(),
                dlogits.data_ptr(), scratch.data_ptr(), _stream(dev)
            ), 'pcm_distill_grad'
        )
        return dlogits, None


def distill_loss(logits, teacher, targets=None, lengths=None, hard_weight=0.0,
                 step_weight=None, status=None):
    """Distillation of ``logits[T,B,V]`` (fp32, bf16 or fp16) from a teacher's
    ``TopLogits`` of shapes [T,B,k]: per row

        (1 - hard_weight) temperature^2 KL(teacher || student)
            + hard_weight * cross entropy(logits, targets)

    with both distributions at the teacher's temperature (1e-3..1e3) over its
    listed tokens and "any other token", summed over steps after weighting step t by
    ``step_weight[t]`` (default: one over the rows with ``lengths > t``), as
    ``DecoderHeadFn`` reduces its cross entropy.  Returns an fp32 scalar that
    carries the gradient of the logits (in fp16 rounded after the incoming
    gradient has gone in, so a loss scale does what it is there for; a
    backward with ``create_graph`` raises, for there is no second derivative).
    Indices outside the vocabulary raise STATUS_BAD_TOKEN in ``status`` (see
    ``check_status``).  Into a graph, forward and backward are captured
    together, while no eager autograd graph of the same leaves is alive."""
    require_device(logits, 'distill logits')
    code = _dtype_code(logits, 'distill logits')
    size = logits.shape
    if len(size) != 3 or 0 in size:
        raise ValueError(
            f'logits have shape {tuple(size)}, expected [T, B, V]'
        )
    steps, batch, vocab = size
    _check_vocab(vocab)
    values, indices, rest, temperature = teacher
    temperature = _check_temperature(temperature)
    if not 1e-3 <= temperature <= 1e3:   # (the loss carries its square)
        raise ValueError(f'temperature {temperature}: expected 1e-3..1e3')
    dev = logits.device
    if indices.dim() != 3 or not 1 <= indices.shape[-1] <= _lib.TOP_MAX:
        raise ValueError(
            f'teacher indices have shape {tuple(indices.shape)}, expected '
            f'[T, B, k] with k in 1..{_lib.TOP_MAX}'
        )
    shape = size[:2]
    listed = shape + indices.shape[-1:]
    values = _operand(values, 'teacher values', dev, listed, *_lib.DTYPES)
    indices = _operand(indices, 'teacher indices', dev, listed, torch.int32)
    if rest is not None:
        rest = _operand(rest, 'teacher rest', dev, shape, torch.float32)
    hard_weight = float(hard_weight)
    if not 0.0 <= hard_weight <= 1.0:
        raise ValueError(f'hard_weight {hard_weight}: expected 0..1')
    if targets is not None:
        targets = _operand(targets, 'targets', dev, shape, torch.int64)
    elif hard_weight > 0:
        raise ValueError('hard_weight needs targets')
    if lengths is not None:
        if lengths.dtype != torch.int32 or lengths.device != dev:
            lengths = lengths.to(device=dev, dtype=torch.int32)
        lengths = _operand(lengths, 'lengths', dev, (batch, ), torch.int32)
    if step_weight is not None:
        step_weight = _operand(
            step_weight.to(device=dev, dtype=torch.float32), 'step_weight',
            dev, (steps, ), torch.float32
        )
    for t in (logits, values, rest, step_weight):
        if _has_tangent(t):
            raise RuntimeError(
                'distill_loss has no derivative in forward mode, and an '
                'operand carries a tangent'
            )
    args = (code, vocab, values, indices, rest, temperature, targets, lengths,
            hard_weight, step_weight, _status_word(status, dev))
    if logits.requires_grad and torch.is_grad_enabled():
        if logits.dtype == torch.float16:
            return DistillHalfLossFn.apply(logits, args)
        return DistillLossFn.apply(logits, args)
    return _distill(logits, False, args)[0]


class BeamStep(NamedTuple):
    """One selection of ``beam_select``: of every batch row's new beams, best
    first, the token i64[W,B], the beam it continues i32[W,B], the score
    f64[W,B] and whether it has ended (bool[W,B], None if beams do not end)."""
    tokens: torch.Tensor
    parents: torch.Tensor
    scores: torch.Tensor
    finished: Optional[torch.Tensor] = None


def beam_select(logits, scores, width=None, temperature=1.0, finished=None,
                end_token=None):
    """One step of a beam search over beams and vocabulary: of the K * V
    candidates ``scores[k, b] + log_softmax(logits[k, b] / temperature)`` of
    every batch row the ``width`` (default K) best, equal ones by beam, then
    token.  ``logits[K,B,V]`` in fp32, bf16 or fp16 (rows k * B + b, the layout
    of the beams' states), ``scores`` f64[K,B] with -inf for a slot that holds
    no beam (at the start: every slot but the first).  ``finished`` bool[K,B]
    with ``end_token``: a finished beam keeps its score and repeats
    ``end_token``.  Returns a ``BeamStep``; ``reorder_states`` lets the states
    follow.  A beam's own tokens are ranked by logit.  No gradient."""
    lib = load()
    require_device(logits, 'beam logits')
    code = _dtype_code(logits, 'beam logits')
    if logits.dim() != 3 or 0 in logits.shape:
        raise ValueError(
            f'logits have shape {tuple(logits.shape)}, expected [K, B, V]'
        )
    beams, batch, vocab = logits.shape
    _check_vocab(vocab)
    temperature = _check_temperature(temperature)
    width = beams if width is None else int(width)
    if not (1 <= beams <= _lib.BEAM_MAX and 1 <= width <= _lib.BEAM_MAX
            and width <= beams * vocab):
        raise ValueError(
            f'{beams} beams and width {width}: expected 1..{_lib.BEAM_MAX}, '
            f'the width within the {beams * vocab} candidates'
        )
    dev = logits.device
    scores = _operand(scores, 'scores', dev, (beams, batch), torch.float64)
    if (finished is None) != (end_token is None):
        raise ValueError('finished and end_token go together')
    finished_out = None
    if finished is not None:
        finished = _operand(finished, 'finished', dev, (beams, batch),
                            torch.bool)
        end_token = int(end_token)
        if not 0 <= end_token < vocab:
            raise ValueError(
                f'end_token {end_token} outside the vocabulary of {vocab}'
            )
        finished_out = torch.empty((width, batch), dtype=torch.bool,
                                   device=dev)
    x2, _, ld = _rows_of(logits.detach(), 'beam logits')
    tokens = torch.empty((width, batch), dtype=torch.int64, device=dev)
    parents = torch.empty((width, batch), dtype=torch.int32, device=dev)
    scores_out = torch.empty((width, batch), dtype=torch.float64, device=dev)
    need = lib.pcm_beam_select_workspace_bytes(beams, batch, vocab, width)
    work = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    with _on(dev):
        check(
            lib.pcm_beam_select(
                x2.data_ptr(), code, ld, scores.data_ptr(), ptr(finished),
                beams, batch, vocab, width, temperature,
                -1 if end_token is None else end_token, tokens.data_ptr(),
                parents.data_ptr(), scores_out.data_ptr(), ptr(finished_out),
                ptr(work), need, _stream(dev)
            ), 'pcm_beam_select'
        )
    return BeamStep(tokens, parents, scores_out, finished_out)


def _state_view(t, row_dim, rows, n):
    """The fields of the pcm_state of state ``n``, a tensor whose dimension
    ``row_dim`` is the beams' rows."""
    dim = t.dim()
    if not -dim <= row_dim < dim:
        raise ValueError(f'state {n}: row dimension {row_dim} of {dim}')
    row_dim %= dim
    shape, size = t.shape, t.element_size()
    if shape[row_dim] != rows:
        raise ValueError(
            f'state {n} has {shape[row_dim]} rows, expected {rows}'
        )
    if t.is_contiguous():
        piece = size * math.prod(shape[row_dim + 1:])
        return (t.data_ptr(), math.prod(shape[:row_dim]), rows * piece, piece,
                piece)
    stride = t.stride()
    inner = 1   # elements of a row's piece, in one stretch
    for d in range(dim - 1, row_dim, -1):
        if shape[d] != 1 and stride[d] != inner:
            raise ValueError(
                f'state {n}: the dimensions after its rows must be contiguous'
            )
        inner *= shape[d]
    outer, outer_stride = 1, 0   # the dimensions before them, as one
    for d in range(row_dim - 1, -1, -1):
        if shape[d] == 1:
            continue
        if outer > 1 and stride[d] != outer * outer_stride:
            raise ValueError(
                f'state {n}: the dimensions before its rows must be evenly '
                'spaced'
            )
        if outer == 1:
            outer_stride = stride[d]
        outer *= shape[d]
    return (t.data_ptr(), outer, outer_stride * size, stride[row_dim] * size,
            inner * size)


def reorder_states(parents, states, row_dims=0, status=None):
    """Lets the states of beams follow them, IN PLACE and in one launch: with
    ``parents`` i32[K,B] (``BeamStep.parents``), row ``k * B + b`` of every
    tensor becomes what its row ``parents[k, b] * B + b`` was.  ``row_dims``:
    the dimension of each tensor that holds the K * B rows, or one for all (the
    StackGRU's hidden [L, K*B, H] has 1, its stack [K*B, D, W] has 0).  Any
    element type; the dimensions after the rows must be contiguous, no two
    tensors may share memory.  A parent outside [0, K) leaves its rows alone
    and raises STATUS_BAD_PARENT in ``status`` (see ``check_status``).  For
    autograd it is an operation in place: a backward that needs a state as it
    was raises."""
    lib = load()
    require_device(parents, 'parents')
    if parents.dtype != torch.int32 or parents.dim() != 2 \
            or 0 in parents.shape:
        raise ValueError('parents: expected int32[K, B]')
    beams, batch = parents.shape
    if beams > _lib.BEAM_MAX:
        raise ValueError(f'{beams} beams: expected 1..{_lib.BEAM_MAX}')
    if isinstance(states, torch.Tensor):
        raise TypeError('states: expected a list of tensors')
    if not 1 <= len(states) <= _lib.MAX_STATES:
        raise ValueError(f'{len(states)} states: expected 1..'
                         f'{_lib.MAX_STATES}')
    if isinstance(row_dims, int):
        row_dims = [row_dims] * len(states)
    if len(row_dims) != len(states):
        raise ValueError('row_dims: one for each state')
    dev = parents.device
    table = []
    for n, (state, row_dim) in enumerate(zip(states, row_dims)):
        if state.device != dev:
            raise ValueError(
                f'state {n} is on {state.device}, the parents on {dev}'
            )
        if state.requires_grad:
            raise ValueError(f'state {n} requires a gradient')
        if _has_tangent(state):
            raise ValueError(f'state {n} carries a tangent')
        table += _state_view(state, row_dim, beams * batch, n)
    if not parents.is_contiguous():
        parents = parents.contiguous()
    _status_word(status, dev)
    with _on(dev):
        check(
            lib.pcm_reorder_states(
                parents.data_ptr(), beams, batch,
                (ctypes.c_int64 * len(table))(*table), len(states),
                ptr(status), _stream(dev)
            ), 'pcm_reorder_states'
        )
    # what an operation saved of them for its backward is no longer there
    torch._C._increment_version(states)


def adam_step(param, grad, exp_avg, exp_avg_sq, lr, beta1, beta2, eps, step,
              grad_scale=1.0):
    """In-place torch.optim.Adam update of a flat fp32 buffer."""
    lib = load()
    require_device(param, 'adam param')
    check(
        lib.pcm_adam_step(
            ptr(param), ptr(grad), ptr(exp_avg), ptr(exp_avg_sq),
            param.numel(), float(lr), float(beta1), float(beta2), float(eps),
            int(step), float(grad_scale), stream_ptr(param.device)
        ), 'pcm_adam_step'
    )
