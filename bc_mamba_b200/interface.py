"""Autograd boundary of the event pipeline, identical in signature to the
reference's Python layer so callers switch without edits:

* ``SelectiveScanFlatChFn`` / ``selective_scan_flat_ch_fn``
  (spike_mamba/selective_scan_interface.py:1015-1237)
* ``RestoreDenseFn`` / ``restore_dense_fn``  (spike_mamba/e_model.py:123-161)
* ``GatherEventsFn`` / ``gather_events``       (spike_mamba/e_model.py:167-193)
* ``extract_events_1d``                        (spike_mamba/e_model.py:361-409)
* ``EventParamsFn`` / ``event_params``          (the parameter transforms of
  Mamba.forward, spike_mamba/e_model.py:210-230, 463, 475-476, in one kernel)

and, without a counterpart there, operators of language models: the gated
linear recurrence (``gated_recurrence``, ``gated_recurrence_step``), the
distillation loss on a teacher's top logits (``distill_topk``,
``distill_topk_with_grad``), token sampling (``sample_tokens``), and the
parts of a linear-attention block: ``decay_attention``,
``decay_attention_step``, ``gated_norm`` and ``add_norm``.

All device work goes through the native shim (``bc_mamba_b200._native``);
there is no Python or CPU fallback.  ``install_shim()`` puts the drop-in
modules ``selective_scan_cuda``, ``extract_events_cuda`` and
``restore_dense_cuda_nodecay`` on ``sys.path`` so the reference's own
``e_model.py`` / ``lra_impl.py`` import them unchanged.
"""
from __future__ import annotations

import contextlib
import sys
from pathlib import Path

import torch

from ._native import load_ops

SHIM_DIR = Path(__file__).resolve().parent / "shim"


def install_shim() -> None:
    """Make ``import selective_scan_cuda`` (and the other two) resolve here."""
    p = str(SHIM_DIR)
    if p not in sys.path:
        sys.path.insert(0, p)


_stage_log = None   # list of (name, start, end) CUDA events while stage_timing() is open


@contextlib.contextmanager
def stage_timing():
    """Record a CUDA event pair on the launching stream around every
    cuda_stage entered while the context is open (autograd's backward thread
    included).  Yields the list of (name, start_event, end_event); read the
    times after a synchronize."""
    global _stage_log
    ops = load_ops()
    prev, _stage_log = _stage_log, []
    ops.time_stages(cuda_stage)           # backward passes in C++ are stages too
    try:
        yield _stage_log
    finally:
        _stage_log = prev
        ops.time_stages(None if prev is None else cuda_stage)


class cuda_stage(contextlib.ContextDecorator):
    """NVTX range named like the reference's profiling stages
    (spike_mamba/runtime_breakdown.py:12-15), timed with CUDA events while
    stage_timing() is open.  A context, or a decorator of functions."""

    def __init__(self, name: str):
        self.name = name

    def _recreate_cm(self):
        return cuda_stage(self.name)      # a decorated function's calls may be nested

    def __enter__(self):
        self.on = torch.cuda.is_available()
        if self.on:
            self.log = _stage_log
            torch.cuda.nvtx.range_push(self.name)
            if self.log is not None:
                self.start = torch.cuda.Event(enable_timing=True)
                self.start.record()

    def __exit__(self, *exc):
        if self.on:
            if self.log is not None:
                end = torch.cuda.Event(enable_timing=True)
                end.record()
                self.log.append((self.name, self.start, end))
            torch.cuda.nvtx.range_pop()
        return False


class SelectiveScanFlatChFn(torch.autograd.Function):
    """Flat per-channel selective scan over event streams.

    Forward inputs (positional): u_flat, k_flat, cu_seqlens, dt_idle,
    dt_active, A, B, C, D, z, max_seqlen, tile_offsets, tile_chunk_size,
    is_depthwise_bc, pw_B, pw_C.  Returns (out, x) where x holds the chunk
    boundary states (non-differentiable); out is gated by silu(z) if z given.
    """

    @staticmethod
    def forward(ctx, u_flat, k_flat, cu_seqlens, dt_idle, dt_active, A, B, C, D, z,
                max_seqlen, tile_offsets, tile_chunk_size, is_depthwise_bc, pw_B, pw_C):
        ops = load_ops()
        u_flat = u_flat.contiguous()
        k_flat = k_flat.contiguous()
        cu_seqlens = cu_seqlens.contiguous()
        dt_idle = dt_idle.contiguous()
        dt_active = dt_active.contiguous()
        A, B, C = A.contiguous(), B.contiguous(), C.contiguous()
        D = D.contiguous() if D is not None else None
        z = z.contiguous() if z is not None else None
        tile_offsets = tile_offsets.contiguous() if tile_offsets is not None else None
        pw_B = pw_B.contiguous() if pw_B is not None else None
        pw_C = pw_C.contiguous() if pw_C is not None else None
        with cuda_stage("sparse_scan_forward"):
            # the forward also keeps the state every 8 events (where the
            # staged kernels run) so the backward does not re-run the recurrence
            res = ops.fwd_flat_ch_ckpt(u_flat, k_flat, cu_seqlens, max_seqlen, dt_idle, dt_active,
                                       A, B, C, D, z, tile_offsets, tile_chunk_size,
                                       is_depthwise_bc, pw_B, pw_C)
        out, x, ckpt = res[0], res[1], res[-1]
        ctx.has_D = D is not None
        ctx.has_z = z is not None
        ctx.has_tiles = tile_offsets is not None
        ctx.has_pw = pw_B is not None
        ctx.max_seqlen = max_seqlen
        ctx.tile_chunk_size = tile_chunk_size
        ctx.is_depthwise_bc = is_depthwise_bc
        saved = [u_flat, k_flat, cu_seqlens, dt_idle, dt_active, A, B, C, x]
        if ctx.has_D:
            saved.append(D)
        if ctx.has_z:
            saved += [z, out]
        if ctx.has_tiles:
            saved.append(tile_offsets)
        if ctx.has_pw:
            saved += [pw_B, pw_C]
        saved.append(ckpt)
        ctx.save_for_backward(*saved)
        ctx.mark_non_differentiable(x)
        # x takes no gradient: without this autograd fills a zero tensor for it
        ctx.set_materialize_grads(False)
        return (res[2] if ctx.has_z else out), x

    @staticmethod
    def backward(ctx, dout, _dx):
        ops = load_ops()
        if dout is None:        # the output was not used in the loss
            return (None,) * 16
        if dout.stride(-1) != 1:
            dout = dout.contiguous()
        it = iter(ctx.saved_tensors)
        u_flat, k_flat, cu_seqlens, dt_idle, dt_active, A, B, C, x = (next(it) for _ in range(9))
        D = next(it) if ctx.has_D else None
        z, out = (next(it), next(it)) if ctx.has_z else (None, None)
        tile_offsets = next(it) if ctx.has_tiles else None
        pw_B, pw_C = (next(it), next(it)) if ctx.has_pw else (None, None)
        ckpt = next(it)
        with cuda_stage("sparse_scan_backward"):
            res = ops.bwd_flat_ch(u_flat, k_flat, cu_seqlens, ctx.max_seqlen, dt_idle, dt_active,
                                  A, B, C, dout, x, D, z, out, tile_offsets,
                                  ctx.tile_chunk_size, ctx.is_depthwise_bc, pw_B, pw_C,
                                  ckpt if ckpt.numel() > 0 else None)
        du, dA, dB, dC, ddt_idle, ddt_active = res[:6]
        rest = iter(res[6:])
        dD = next(rest) if ctx.has_D else None
        dz = next(rest) if ctx.has_z else None
        dpw_B, dpw_C = (next(rest), next(rest)) if ctx.has_pw else (None, None)
        return (du, None, None, ddt_idle, ddt_active, dA, dB, dC, dD, dz,
                None, None, None, None, dpw_B, dpw_C)


def selective_scan_flat_ch_fn(u_flat, k_flat, cu_seqlens, max_seqlen, dt_idle, dt_active, A, B, C,
                              D=None, z=None, tile_offsets=None, tile_chunk_size=0,
                              is_depthwise_bc=False, pw_B=None, pw_C=None):
    """Autograd-enabled flat per-channel selective scan; returns (out, x)."""
    return SelectiveScanFlatChFn.apply(u_flat, k_flat, cu_seqlens, dt_idle, dt_active, A, B, C,
                                       D, z, max_seqlen, tile_offsets, tile_chunk_size,
                                       is_depthwise_bc, pw_B, pw_C)


class RestoreDenseFn(torch.autograd.Function):
    """Zero-order-hold restore: (E,) event values -> (B, L, D) dense."""

    @staticmethod
    def forward(ctx, y_flat, time_steps_i32, cu_seqlens, dim: int, seqlen: int, base_mask=None, expand: int = 1):
        # the forward also writes the event bitmap (one bit per channel and
        # position) that the backward sweeps instead of the event times;
        # base_mask: the extraction's threshold mask of this stream, which the
        # bitmap is transposed from instead
        with cuda_stage("dense_restoration_forward"):
            out, bitmap = load_ops().restore_dense_fwd_bitmap(y_flat, time_steps_i32, cu_seqlens, dim, seqlen,
                                                              base_mask=base_mask, expand=expand)
        ctx.save_for_backward(time_steps_i32, cu_seqlens, bitmap)
        ctx.dim = dim
        ctx.seqlen = seqlen
        return out

    @staticmethod
    def backward(ctx, dout):
        time_steps_i32, cu_seqlens, bitmap = ctx.saved_tensors
        with cuda_stage("restore_backward"):
            dy = load_ops().restore_dense_bwd_bitmap(dout.contiguous(), time_steps_i32, cu_seqlens, bitmap,
                                                     ctx.dim, ctx.seqlen)
        return dy, None, None, None, None, None, None


# the bitmap of the restore holds at most this many events per channel; up to
# it the extraction's mask gives the same bitmap
MASK_RESTORE_MAX_SEQLEN = 4095


def restore_dense_fn(y_flat, time_steps_i32, cu_seqlens, dim: int, seqlen: int, base_mask=None, expand: int = 1):
    """base_mask (optional): the mask buffer extract_events_1d(...,
    return_mask=True) returned for this stream (seqlen <= 4095)."""
    return RestoreDenseFn.apply(y_flat, time_steps_i32, cu_seqlens, dim, seqlen, base_mask, int(expand))


class EventParamsFn(torch.autograd.Function):
    """An event block's parameter transforms in one launch each way
    (spike_mamba/e_model.py:463 A = -exp(A_log); :475-476 W_B, W_C = the
    halves of W_BC; :210-230 dt_idle / dt_active = softplus(a0 / a1) + eps):
    the same values and gradients as those PyTorch ops, with one kernel and
    one autograd node instead of eight of each."""

    @staticmethod
    def forward(ctx, A_log, W_BC, a0, a1, eps: float):
        A, W_B, W_C, dt_idle, dt_active = load_ops().event_params_fwd(A_log, W_BC, a0, a1, float(eps))
        ctx.save_for_backward(A, a0, a1)
        ctx.set_materialize_grads(False)   # an output without a gradient reaches the kernel as NULL
        return A, W_B, W_C, dt_idle, dt_active

    @staticmethod
    def backward(ctx, dA, dW_B, dW_C, ddt_idle, ddt_active):
        A, a0, a1 = ctx.saved_tensors
        c = lambda t: None if t is None else t.contiguous()
        dA_log, dW_BC, da0, da1 = load_ops().event_params_bwd(A, a0, a1, c(dA), c(dW_B), c(dW_C), c(ddt_idle),
                                                              c(ddt_active))
        return dA_log, dW_BC, da0, da1, None


def event_params(A_log, W_BC, a0, a1, eps: float = 1e-6):
    """(A, W_B, W_C, dt_idle, dt_active) of one event block's parameters."""
    return EventParamsFn.apply(A_log, W_BC, a0, a1, eps)


class GatherEventsFn(torch.autograd.Function):
    """u_flat[e] = x_conv[b, d, t] at (channel_ids[e] = b*D + d, time_steps[e])."""

    @staticmethod
    def forward(ctx, x_conv, channel_ids_i32, time_steps_i32, cu_seqlens=None):
        x_c = x_conv.contiguous()
        with cuda_stage("active_gather_forward"):
            out_x = load_ops().gather_events_fwd(x_c, channel_ids_i32, time_steps_i32)[0]
        # with the extraction's cu_seqlens the backward reads each channel's
        # rows from it instead of recovering them from channel_ids
        if cu_seqlens is not None:
            ctx.save_for_backward(channel_ids_i32, time_steps_i32, cu_seqlens)
        else:
            ctx.save_for_backward(channel_ids_i32, time_steps_i32)
        ctx.shape = x_c.shape
        return out_x

    @staticmethod
    def backward(ctx, grad_x):
        saved = ctx.saved_tensors
        channel_ids_i32, time_steps_i32 = saved[0], saved[1]
        B, D, L = ctx.shape
        with cuda_stage("gather_scatter_backward"):
            if len(saved) == 3:
                dx = load_ops().gather_events_bwd_rows(grad_x.contiguous(), time_steps_i32, saved[2], B * D, L)
            else:
                dx = load_ops().gather_events_bwd(grad_x.contiguous(), channel_ids_i32,
                                                  time_steps_i32, B * D, L)[0]
        return dx.view(B, D, L), None, None, None


class ConvEventsFn(torch.autograd.Function):
    """silu(causal depthwise conv1d(x) + bias) evaluated only at the events:
    replaces the dense ``x_conv = act(conv1d(x))[..., :L]`` of Mamba.forward
    followed by ``GatherEventsFn`` (spike_mamba/e_model.py:442-451, 404-406),
    whose result is read nowhere else.  ``weight`` is the conv1d weight
    ([D, 1, K] or [D, K]); ``cu_seqlens`` must describe the stream (events of a
    channel contiguous and time-ordered, as extraction produces them)."""

    @staticmethod
    def forward(ctx, x, weight, bias, channel_ids_i32, time_steps_i32, cu_seqlens):
        with cuda_stage("active_gather_forward"):
            u_flat = load_ops().conv_events_fwd(x, weight, bias, channel_ids_i32, time_steps_i32)[0]
        ctx.save_for_backward(x, weight, bias if bias is not None else torch.empty(0), time_steps_i32,
                              cu_seqlens)
        ctx.has_bias = bias is not None
        return u_flat

    @staticmethod
    def backward(ctx, grad_u):
        x, weight, bias, time_steps_i32, cu_seqlens = ctx.saved_tensors
        with cuda_stage("gather_scatter_backward"):
            dx, dw, db = load_ops().conv_events_bwd(x, weight, bias if ctx.has_bias else None,
                                                    time_steps_i32, cu_seqlens, grad_u.contiguous())
        dw = dw.view(weight.shape).to(weight.dtype)
        db = db.to(bias.dtype) if ctx.has_bias else None
        return dx, dw, db, None, None, None


def conv_events(x, weight, bias, channel_ids_i32, time_steps_i32, cu_seqlens):
    return ConvEventsFn.apply(x, weight, bias, channel_ids_i32, time_steps_i32, cu_seqlens)


class ExtractGatherFn(torch.autograd.Function):
    """Extraction + expansion + gather of x_conv in one fill pass: the
    forward of extract_base_events -> expand_base_events -> GatherEventsFn
    (reference spike_mamba/e_model.py:371-390, 167-193) with the same outputs;
    only x_flat is differentiable (w.r.t. x_conv), and its backward is the
    gather backward from the stream's rows."""

    @staticmethod
    def forward(ctx, x_conv, spikes, threshold, expand, bld, max_out, keep_mask):
        x_c = x_conv.contiguous()
        # threshold: one float, or a tensor with one threshold per feature
        ft = threshold if isinstance(threshold, torch.Tensor) else None
        with cuda_stage("routing_index_extraction"):
            # the maximum count arrives on the host with the event total (one
            # synchronisation); expansion copies counts, so it is max_seqlen
            # of the expanded stream too
            res, max_seqlen = load_ops().extract_expanded_events(
                spikes, 0.0 if ft is not None else threshold, expand, bld=bld, x_conv=x_c, feature_thresholds=ft,
                keep_mask=keep_mask)
        ch, ts, kf, cu, _mx, x_flat = res[:6]
        max_out.append(int(max_seqlen))
        ctx.save_for_backward(ts, cu)
        ctx.shape = x_c.shape
        ctx.mark_non_differentiable(ch, ts, kf, cu, *res[6:])
        ctx.set_materialize_grads(False)
        # keep_mask: also the buffer holding the threshold mask (restore_dense_fn's base_mask)
        return (x_flat, ch, ts, kf, cu, res[6]) if keep_mask else (x_flat, ch, ts, kf, cu)

    @staticmethod
    def backward(ctx, grad_x, *_):
        if grad_x is None:
            return (None,) * 7
        ts, cu = ctx.saved_tensors
        B, D, L = ctx.shape
        with cuda_stage("gather_scatter_backward"):
            dx = load_ops().gather_events_bwd_rows(grad_x.contiguous(), ts, cu, B * D, L)
        return dx.view(B, D, L), None, None, None, None, None, None


def gather_events(x_conv, channel_ids_i32, time_steps_i32, cu_seqlens=None):
    """cu_seqlens (optional): the stream's channel offsets when it is in
    extraction order, as extraction returns it."""
    return GatherEventsFn.apply(x_conv, channel_ids_i32, time_steps_i32, cu_seqlens)


def extract_events_base(base_input, x_conv, threshold: float, expand: int):
    """Extraction from the (B, d_model, L) layout extract_base_events takes
    (what Mamba.extract_events_1d builds by transposing hidden_states), then
    expansion and the gather of x_conv (B, D, L).

    Returns (channel_ids, time_steps, k_flat, cu_seqlens, max_seqlen, x_conv_flat).
    """
    # extraction, expansion and the gather of x_conv in one fill pass (the
    # base stream is never written)
    mx = []
    x_flat, ch, ts, kf, cu = ExtractGatherFn.apply(x_conv, base_input.contiguous(), float(threshold), int(expand),
                                                   False, mx, False)
    return ch, ts, kf, cu, mx[0], x_flat


def extract_events_1d(hidden_states, x_conv, threshold, expand: int, return_mask: bool = False):
    """Threshold (B, L, d_model) spikes into the expanded event stream and
    gather x_conv (B, D, L) at the events, like Mamba.extract_events_1d.
    `threshold` is a float as in the reference, or a contiguous float32
    (d_model,) tensor on the spikes' device: feature j fires above
    threshold[j].

    Returns (channel_ids, time_steps, k_flat, cu_seqlens, max_seqlen, x_conv_flat), and with
    return_mask=True also the buffer holding the threshold mask (for
    restore_dense_fn's base_mask).
    """
    # straight from the (B, L, d_model) layout (the reference first makes a
    # transposed (B, d_model, L) copy, e_model.py:376); extraction, expansion
    # and the gather of x_conv in one fill pass, the maximum count back with
    # the event total (one synchronisation, no .item())
    mx = []
    thr = threshold if isinstance(threshold, torch.Tensor) else float(threshold)
    outs = ExtractGatherFn.apply(x_conv, hidden_states.contiguous(), thr, int(expand), True, mx, bool(return_mask))
    x_flat, ch, ts, kf, cu = outs[:5]
    if return_mask:
        return ch, ts, kf, cu, mx[0], x_flat, outs[5]
    return ch, ts, kf, cu, mx[0], x_flat


class EventDecoder:
    """The event path one token at a time, in place of Mamba.step
    (reference spike_mamba/e_model.py:508-568, which reads self.pw_B /
    self.pw_C that Mamba does not define).  Each step runs extraction's
    compare on the token's spikes, the depthwise scan update of the channels
    that fire and the restore's hold, so decoding a sequence gives exactly the
    outputs extract_events_* -> selective_scan_flat_ch_fn (depthwise) ->
    restore_dense_fn give for it.  With kernel_size > 0 the token's x is the
    conv input and passes the causal depthwise conv + SiLU first (the
    conv_state of e_model.py:512-518, kept here).

    State per channel (B*D of them): eta [B*D, N] (normalised scan state),
    counters [B*D, 2] (tokens since the last event, events so far), held
    [B*D] (latest output), conv_state [B, D, K]."""

    def __init__(self, batch: int, dim: int, dstate: int, device, dtype=torch.float32, kernel_size: int = 0):
        nc = batch * dim
        self.eta = torch.zeros(nc, dstate, dtype=torch.float32, device=device)
        self.counters = torch.zeros(nc, 2, dtype=torch.int32, device=device)
        self.held = torch.zeros(nc, dtype=torch.float32, device=device)
        self.conv_state = (torch.zeros(batch, dim, kernel_size, dtype=dtype, device=device)
                           if kernel_size > 0 else None)

    def step(self, x, spikes, threshold: float, dt_idle, dt_active, A, W_B, W_C, D=None,
             conv_weight=None, conv_bias=None):
        """x [B, D] (u, or the conv input with a conv state), spikes [B, d_model]
        -> y [B, D].  W_B / W_C are the effective [D, N] weights."""
        return load_ops().event_decode_step(x.contiguous(), spikes.contiguous(), float(threshold),
                                            dt_idle.contiguous(), dt_active.contiguous(), A, W_B.contiguous(),
                                            W_C.contiguous(), D, self.eta, self.counters, self.held,
                                            self.conv_state, conv_weight, conv_bias)


# ------------------------------------------------ language-model operators ----
# (no counterpart in the reference: a sequence mixer, a training loss and a
# token sampler for models built on this package's scans; their autograd
# functions are C++, in the shim, and their gradients not differentiable)


def gated_recurrence(x, r, i, lam, h0=None, cu_seqlens=None, decay_scale: float = 8.0):
    """h_t = a_t h_(t-1) + sqrt(1 - a_t^2) sigmoid(i_t) x_t with the decay
    a_t = exp(-decay_scale softplus(lam) sigmoid(r_t)), per feature.

    x (values), r (decay gate) and i (input gate) are (B, L, D), or packed
    (T, D) with cu_seqlens (n + 1,) int32, ascending from 0 to T (sequences may
    be empty); float32, float16 or bfloat16, any batch and position strides.
    lam (D,) and the entering states h0 (B, D) (None: zeros) are float32.
    Returns (y, h_last): y = h in x's dtype, and the float32 states after each
    sequence's last token, which continue it as h0 of a next call or as the
    state of gated_recurrence_step.  Differentiable in x, r, i, lam and h0; the
    state is float32 throughout and gradients are the same from run to run."""
    with cuda_stage("gated_recurrence_forward"):
        return load_ops().gated_recurrence(x, r, i, lam, h0, cu_seqlens, decay_scale)


def gated_recurrence_step(x, r, i, lam, h, decay_scale: float = 8.0):
    """One token of gated_recurrence for every sequence: x, r, i (B, D), the
    state h (B, D) float32 contiguous, updated in place.  Returns y (B, D).  No
    gradient passes through it: while gradients are recorded, inputs that
    require them are refused, and a graph that saved h finds it modified."""
    return load_ops().gated_rec_step(x, r, i, lam, h, decay_scale)


def decay_attention(q, k, v, log_decay, h0=None, cu_seqlens=None):
    """Linear attention with a decay for each head: with a_t = exp(log_decay_t),
    S_t = a_t S_(t-1) + k_t v_t^T (N x P) and y_t = S_t^T q_t.

    v (B, L, H, P), q and k (B, L, Hk, N), or packed (T, ..) with cu_seqlens
    (n + 1,) int32, ascending from 0 (sequences may be empty; rows behind the
    last one have y and gradients 0); float32, float16 or bfloat16, any strides
    of the batch, the tokens and the heads.  Hk divides H: head h reads query
    and key h // (H / Hk); N is 128 at most.  log_decay is float32, at most 0
    (-inf drops the state): one per token and head (B, L, H) (packed (T, H)),
    or one constant for each head (H,).  The entering states h0 (B, H, N, P)
    (None: zeros) are float32.
    Returns (y, h_last): y in v's dtype, and the float32 states after each
    sequence's last token, which continue it as h0 of a next call or as the
    states of decay_attention_step.  Differentiable in q, k, v, log_decay and
    h0; gradients are the same from run to run.  States are float32; products
    run on the tensor cores with float32 sums, of operands as sums of bfloat16
    numbers: float16 inputs as two and float32 ones as three, which hold them
    exactly, what is computed between them as two where a result ends in 16 bits
    (within 2^-17) and three where it ends in float32; products of two of these
    parts that lie below 2^-16 or, for float32 results, 2^-24 of the whole are
    left out.  A dense call of up to four tokens that records no gradient sums in
    float32 throughout: its y may differ in the last bit from that of a call that
    does.
    A value that is not finite reaches no token before its own (behind it, what
    would be infinite may be NaN); the 64 tokens around it take longer, 0.2 ms
    forward and 2 ms backward."""
    with cuda_stage("decay_attention_forward"):
        return load_ops().decay_attention(q, k, v, log_decay, h0, cu_seqlens)


def decay_attention_step(q, k, v, log_decay, h):
    """One token of decay_attention for every sequence: v (B, H, P), q and k
    (B, Hk, N), log_decay (B, H) or (H,), the states h (B, H, N, P) float32
    contiguous, updated in place.  Returns y (B, H, P).  No gradient passes
    through it, as in gated_recurrence_step."""
    return load_ops().decay_attn_step(q, k, v, log_decay, h)


def gated_norm(x, gate, weight, groups: int = 1, eps: float = 1e-6):
    """The norm of a mixer's output with its gate, per row of x (.., D) and
    group of D / groups features (a head each, 8192 features at most):
    x / sqrt(mean(x^2) + eps) * weight * silu(gate).  gate has the shape and
    dtype of x (float32, float16 or bfloat16, any row stride), weight (D,) is
    float32.  Differentiable in all three; sums are float32, in a fixed order."""
    with cuda_stage("gated_norm_forward"):
        return load_ops().gated_norm(x, gate, weight, groups, eps)


def add_norm(residual, branch, weight, scale=None, eps: float = 1e-6):
    """The residual addition of a block's output and the norm before the next
    block: v = residual + scale * branch, normed = v / sqrt(mean(v^2) + eps) *
    weight, over the last dimension (8192 at most).  branch (.., D) is float32,
    float16 or bfloat16, residual of its dtype or float32, weight and scale (D,)
    (None: 1) float32.  Returns (v in residual's dtype, normed in branch's); the
    norm is that of v before it is rounded.  Differentiable in all."""
    with cuda_stage("add_norm_forward"):
        return load_ops().add_norm(residual, branch, weight, scale, eps)


def distill_topk(logits, teacher_logits, teacher_ids, weight=None, temperature: float = 1.0):
    """Per-row loss weight tau^2 KL(teacher || student), tau the temperature:
    the teacher's softmax over its K top logits (T, K) with token ids (T, K)
    (int32 or int64; K up to 1024) against the student's softmax over the whole
    vocabulary, logits (T, V) in float32, float16 or bfloat16.  Entries whose
    id lies outside [0, V) or whose logit is -inf are absent (lists may end
    early); a row without entries, or of weight 0, has loss and gradient 0
    whatever its logits hold.  weight (T,) float32.  Differentiable in logits.
    Returns the losses (T,) float32."""
    with cuda_stage("distill_forward"):
        return load_ops().distill_topk(logits, teacher_logits, teacher_ids, weight, temperature)


def distill_topk_with_grad(logits, teacher_logits, teacher_ids, weight=None, temperature: float = 1.0):
    """distill_topk and its gradient in one call: (loss (T,), dlogits (T, V)),
    dlogits for an upstream gradient of one per row (put a mean's 1/T, or a loss
    scale, into weight).  It reads the logits from memory once where the
    autograd pair reads them twice."""
    with torch.no_grad(), cuda_stage("distill_forward"):
        loss, _, dz = load_ops().distill_fwd(logits, teacher_logits, teacher_ids, weight, temperature, True)
    return loss, dz


def _per_row(value, off, dtype):
    """A setting as (number of every row, tensor of one per row or None)."""
    if not isinstance(value, torch.Tensor):
        return (off if value is None else value), None
    if dtype == torch.int32 and value.dtype != dtype:
        # (in a type that holds both ends; a NaN is off, as in the other settings)
        wide = value.double().nan_to_num(0.0) if value.is_floating_point() else value.to(torch.int64)
        value = wide.clamp(0, 2 ** 31 - 1)
    return off, value if value.dtype == dtype else value.to(dtype)


def sample_tokens(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One token per row of logits (B, V) from given uniform numbers u (B,) in
    [0, 1), with temperature, top-k, top-p and min-p, each a number or a tensor
    of one per row.  Filters apply in that order: top-p to the mass that top-k
    leaves, min-p relative to the most likely token.  temperature <= 0 is greedy,
    top_k <= 0, top_p >= 1 and min_p <= 0 are off; ties go to the lowest index.
    Probabilities are summed as integers, so the token depends on logits, u and
    the settings alone.  Returns (tokens (B,) int64, log-probabilities among the
    kept tokens (B,) float32); a row whose logits are all -inf or NaN gives token
    -1 and log-probability -inf."""
    t, ts = _per_row(temperature, 1.0, torch.float32)
    k, ks = _per_row(top_k, 0, torch.int32)
    p, ps = _per_row(top_p, 1.0, torch.float32)
    m, ms = _per_row(min_p, 0.0, torch.float32)
    with torch.no_grad(), cuda_stage("sample_tokens"):
        tokens, logprob = load_ops().sample_tokens(logits, u, t, k, p, m, ts, ks, ps, ms)
    return tokens, logprob
