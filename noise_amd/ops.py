"""torch.library registrations of the drop-ins, so the reference's torch.compile'd callers trace through them
without graph breaks: population_loss is compiled at eggroll.py:115, head_loss, block_forward and
coordinate_differences at run.py:89, 102, 120, and attention sits inside the compiled forwards
(utils/model.py:14, 95). Fake implementations give output shapes and dtypes; the real ones call libnoise_amd.

  torch.ops.noise_amd.attention(q, k, v, window)                      utils/model.py:24
  torch.ops.noise_amd.lowrank(x, weight, a, b, sign, dir_div)         eggroll.py:56
  torch.ops.noise_amd.lowrank_embed(weight, a, b, idx, sign, dir_div) eggroll.py:61
  torch.ops.noise_amd.population_loss(names, params, noise_a, noise_b, sign, idx, targets, n_layer,
                                      dir_div, fp32_head)             eggroll.py:66
  torch.ops.noise_amd.head_loss(x, weight, targets, vocab)            run.py:90
  torch.ops.noise_amd.block_forward(x, w, ve, cos, sin, window, o, attn, fc, mlp)   run.py:103
  torch.ops.noise_amd.coordinate_differences(raw, y, sigma)           run.py:121

Ops take flat tensor lists where the reference passes dicts: population_loss's parameter and noise dicts
become one list per field in the order of `names` (newline-separated parameter names), with the noise of
a 1-D parameter (the mixing scalars' eps) in noise_a and None in noise_b; block_forward's weight dict is
the list (q, k, v, gate or None, proj, fc, out). The reference-signature wrappers that pack them are
noise_amd.eggroll.population_loss and noise_amd.dust.head_loss / block_forward / coordinate_differences.
"""
from typing import List, Optional, Tuple

import torch
from torch import Tensor
from torch.autograd import forward_ad
from torch.library import custom_op

from . import clip as _clip
from . import distill as _distill
from . import dust, eggroll, model
from . import residual as _residual
from . import sinks as _sinks
from . import vocab as _vocab

BLOCK_WEIGHTS = ('q', 'k', 'v', 'gate', 'proj', 'fc', 'out')


@custom_op('noise_amd::attention', mutates_args=())
def attention(q: Tensor, k: Tensor, v: Tensor, window: int) -> Tensor:
    return model.attention(q, k, v, window)


@attention.register_fake
def _attention_fake(q, k, v, window):
    return q.new_empty(q.shape)


@custom_op('noise_amd::lowrank', mutates_args=())
def lowrank(x: Tensor, weight: Tensor, a: Tensor, b: Tensor, sign: Tensor, dir_div: int) -> Tensor:
    return eggroll.lowrank_eager(x, weight, a, b, sign, dir_div=dir_div)


@lowrank.register_fake
def _lowrank_fake(x, weight, a, b, sign, dir_div):
    return x.new_empty((x.shape[0], x.shape[1], weight.shape[0]), dtype=torch.float32)


@custom_op('noise_amd::lowrank_embed', mutates_args=())
def lowrank_embed(weight: Tensor, a: Tensor, b: Tensor, idx: Tensor, sign: Tensor, dir_div: int) -> Tensor:
    return eggroll.lowrank_embed_eager(weight, a, b, idx, sign, dir_div=dir_div)


@lowrank_embed.register_fake
def _lowrank_embed_fake(weight, a, b, idx, sign, dir_div):
    return weight.new_empty((sign.shape[0], idx.shape[0], weight.shape[1]), dtype=torch.float32)


@custom_op('noise_amd::population_loss', mutates_args=())
def population_loss(names: str, params: List[Tensor], noise_a: List[Optional[Tensor]],
                    noise_b: List[Optional[Tensor]], sign: Tensor, idx: Tensor, targets: Tensor, n_layer: int,
                    dir_div: int, fp32_head: bool) -> Tensor:
    keys = names.split('\n')
    if not (len(keys) == len(params) == len(noise_a) == len(noise_b)):
        raise ValueError(f'population_loss: {len(keys)} names for {len(params)} parameters, '
                         f'{len(noise_a)} / {len(noise_b)} noise entries')
    p = dict(zip(keys, params))
    noise = {}
    for k, a, b in zip(keys, noise_a, noise_b):
        if a is not None:
            noise[k] = a if b is None else (a, b)
    return eggroll.population_loss_eager(p, noise, sign, idx, targets, n_layer=n_layer, dir_div=dir_div,
                                         fp32_head=fp32_head)


@population_loss.register_fake
def _population_loss_fake(names, params, noise_a, noise_b, sign, idx, targets, n_layer, dir_div, fp32_head):
    return sign.new_empty((sign.shape[0],), dtype=torch.float32)


@custom_op('noise_amd::head_loss', mutates_args=())
def head_loss(x: Tensor, weight: Tensor, targets: Tensor, vocab: int) -> Tensor:
    return dust.head_loss_eager(x, weight, targets, vocab)


@head_loss.register_fake
def _head_loss_fake(x, weight, targets, vocab):
    return x.new_empty((targets.numel(),), dtype=torch.float32)


@custom_op('noise_amd::block_forward', mutates_args=())
def block_forward(x: Tensor, w: List[Optional[Tensor]], ve: Optional[Tensor], cos: Tensor, sin: Tensor, window: int,
                  o: Optional[Tensor], attn: Optional[Tensor], fc: Optional[Tensor],
                  mlp: Optional[Tensor]) -> Tensor:
    if len(w) != len(BLOCK_WEIGHTS):
        raise ValueError(f'block_forward: expected the weights {BLOCK_WEIGHTS}, got {len(w)} tensors')
    return dust.block_forward_eager(x, dict(zip(BLOCK_WEIGHTS, w)), ve, cos, sin, window, o, attn, fc, mlp)


@block_forward.register_fake
def _block_forward_fake(x, w, ve, cos, sin, window, o, attn, fc, mlp):
    return x.new_empty(x.shape, dtype=torch.float32)


@custom_op('noise_amd::coordinate_differences', mutates_args=())
def coordinate_differences(raw: Tensor, y: Tensor, sigma: float) -> Tensor:
    return dust.head_error(raw, y, raw.shape[-1], sigma)


@coordinate_differences.register_fake
def _coordinate_differences_fake(raw, y, sigma):
    return raw.new_empty(raw.shape, dtype=torch.float32)


# --- operators with gradients ---
# (an absent gradient of an optional tensor leaves the backward operators as an empty tensor; sink_attention always computes what
# its backward pass needs, sink_attention_output never does)


def _backwards_only(name):
    """Refuses an operator's call inside a forward-mode level. torch.func.jvp hands an operator plain tensors: whether they
    carry tangents cannot be told here, and those that do would get derivatives of 0."""
    if forward_ad._current_level >= 0:
        raise NotImplementedError(f'torch.ops.noise_amd.{name}: forward-mode derivatives are not implemented')


@custom_op('noise_amd::qk_norm_rotary', mutates_args=())
def qk_norm_rotary(q: Tensor, k: Tensor, cos: Tensor, sin: Tensor, q_weight: Optional[Tensor],
                   k_weight: Optional[Tensor], start: Optional[Tensor], eps: float) -> Tuple[Tensor, Tensor]:
    _backwards_only('qk_norm_rotary')
    return _sinks.norm_forward(q, k, cos, sin, q_weight, k_weight, start, eps)


@qk_norm_rotary.register_fake
def _qk_norm_rotary_fake(q, k, cos, sin, q_weight, k_weight, start, eps):
    return q.new_empty(q.shape), k.new_empty(k.shape)


@custom_op('noise_amd::qk_norm_rotary_backward', mutates_args=())
def qk_norm_rotary_backward(dq: Tensor, dk: Tensor, q: Tensor, k: Tensor, cos: Tensor, sin: Tensor,
                            q_weight: Optional[Tensor], k_weight: Optional[Tensor], start: Optional[Tensor],
                            eps: float) -> Tuple[Tensor, Tensor, Tensor, Tensor]:
    _backwards_only('qk_norm_rotary_backward')
    grads = _sinks.norm_backward(dq, dk, q, k, cos, sin, q_weight, k_weight, start, eps)
    return tuple(q.new_empty(0) if g is None else g for g in grads)


@qk_norm_rotary_backward.register_fake
def _qk_norm_rotary_backward_fake(dq, dk, q, k, cos, sin, q_weight, k_weight, start, eps):
    return (q.new_empty(q.shape), k.new_empty(k.shape),
            *(q.new_empty(0) if w is None else w.new_empty(w.shape) for w in (q_weight, k_weight)))


def _qk_norm_rotary_setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs[:7])
    ctx.eps = inputs[7]


def _qk_norm_rotary_backward(ctx, dq, dk):
    q, k, cos, sin, qw, kw, start = ctx.saved_tensors
    dq, dk, dqw, dkw = torch.ops.noise_amd.qk_norm_rotary_backward(dq, dk, q, k, cos, sin, qw, kw, start, ctx.eps)
    return dq, dk, None, None, None if qw is None else dqw, None if kw is None else dkw, None, None


qk_norm_rotary.register_autograd(_qk_norm_rotary_backward, setup_context=_qk_norm_rotary_setup)


@custom_op('noise_amd::qk_norm_rotary_append', mutates_args=('k_cache', 'v_cache'))
def qk_norm_rotary_append(q: Tensor, k: Tensor, v: Tensor, cos: Tensor, sin: Tensor, k_cache: Tensor, v_cache: Tensor,
                          start: Tensor, q_weight: Optional[Tensor], k_weight: Optional[Tensor], eps: float) -> Tensor:
    _backwards_only('qk_norm_rotary_append')
    return _sinks.qk_norm_rotary_append(q, k, v, cos, sin, k_cache, v_cache, start, q_weight, k_weight, eps)


@qk_norm_rotary_append.register_fake
def _qk_norm_rotary_append_fake(q, k, v, cos, sin, k_cache, v_cache, start, q_weight, k_weight, eps):
    return q.new_empty(q.shape)


@custom_op('noise_amd::sink_attention', mutates_args=())
def sink_attention(q: Tensor, k: Tensor, v: Tensor, window: int, sinks: int,
                   lengths: Optional[Tensor]) -> Tuple[Tensor, Tensor, Tensor]:
    _backwards_only('sink_attention')
    return _sinks.attend_forward(q, k, v, window, sinks, lengths, True)


@sink_attention.register_fake
def _sink_attention_fake(q, k, v, window, sinks, lengths):
    return q.new_empty(q.shape), q.new_empty(q.shape), q.new_empty((q.shape[0], q.shape[2], q.shape[1]), dtype=torch.float32)


@custom_op('noise_amd::sink_attention_output', mutates_args=())
def sink_attention_output(q: Tensor, k: Tensor, v: Tensor, window: int, sinks: int, lengths: Optional[Tensor]) -> Tensor:
    """sink_attention's output alone, without what its backward pass needs"""
    _backwards_only('sink_attention_output')
    return _sinks.attend_forward(q, k, v, window, sinks, lengths, False)[0]


@sink_attention_output.register_fake
def _sink_attention_output_fake(q, k, v, window, sinks, lengths):
    return q.new_empty(q.shape)


@custom_op('noise_amd::sink_attention_backward', mutates_args=())
def sink_attention_backward(dout: Tensor, q: Tensor, k: Tensor, v: Tensor, out: Tensor, rest: Tensor, lse: Tensor,
                            window: int, sinks: int, lengths: Optional[Tensor]) -> Tuple[Tensor, Tensor, Tensor]:
    _backwards_only('sink_attention_backward')
    return tuple(_sinks.attend_backward(dout, q, k, v, out, rest, lse, window, sinks, lengths))


@sink_attention_backward.register_fake
def _sink_attention_backward_fake(dout, q, k, v, out, rest, lse, window, sinks, lengths):
    return tuple(t.new_empty(t.shape) for t in (q, k, v))


def _sink_attention_setup(ctx, inputs, output):
    q, k, v, ctx.window, ctx.sinks, lengths = inputs
    ctx.mark_non_differentiable(*output[1:])
    ctx.save_for_backward(q, k, v, *output, lengths)


def _sink_attention_backward(ctx, dout, *_):
    *saved, lengths = ctx.saved_tensors
    return (*torch.ops.noise_amd.sink_attention_backward(dout, *saved, ctx.window, ctx.sinks, lengths),
            None, None, None)


sink_attention.register_autograd(_sink_attention_backward, setup_context=_sink_attention_setup)


@custom_op('noise_amd::sink_attention_decode', mutates_args=())
def sink_attention_decode(q: Tensor, k_cache: Tensor, v_cache: Tensor, start: Tensor, window: int,
                          sinks: int) -> Tensor:
    _backwards_only('sink_attention_decode')
    return _sinks.sink_attention_decode(q, k_cache, v_cache, start, window, sinks)


@sink_attention_decode.register_fake
def _sink_attention_decode_fake(q, k_cache, v_cache, start, window, sinks):
    return q.new_empty(q.shape)


@custom_op('noise_amd::distill_loss', mutates_args=())
def distill_loss(logits: Tensor, teacher_logits: Tensor, teacher_index: Tensor, vocab: int, temperature: float,
                 softcap: Optional[float]) -> Tensor:
    _backwards_only('distill_loss')
    return _distill.distill('distill_loss', logits, teacher_logits, teacher_index, None, vocab, temperature, softcap,
                           False)[0]


@distill_loss.register_fake
def _distill_loss_fake(logits, teacher_logits, teacher_index, vocab, temperature, softcap):
    return logits.new_empty(logits.shape[:-1], dtype=torch.float32)


@custom_op('noise_amd::distill_loss_grad', mutates_args=())
def distill_loss_grad(logits: Tensor, teacher_logits: Tensor, teacher_index: Tensor, weight: Optional[Tensor],
                      vocab: int, temperature: float, softcap: Optional[float]) -> Tuple[Tensor, Tensor]:
    _backwards_only('distill_loss_grad')
    return _distill.distill('distill_loss_grad', logits, teacher_logits, teacher_index, weight, vocab, temperature,
                           softcap, True)


@distill_loss_grad.register_fake
def _distill_loss_grad_fake(logits, teacher_logits, teacher_index, weight, vocab, temperature, softcap):
    return logits.new_empty(logits.shape[:-1], dtype=torch.float32), logits.new_empty(logits.shape)


def _distill_loss_setup(ctx, inputs, output):
    logits, teacher_logits, teacher_index, *ctx.more = inputs
    ctx.save_for_backward(logits, teacher_logits, teacher_index)


def _distill_loss_backward(ctx, weight):
    return (torch.ops.noise_amd.distill_loss_grad(*ctx.saved_tensors, weight, *ctx.more)[1], None, None, None, None, None)


distill_loss.register_autograd(_distill_loss_backward, setup_context=_distill_loss_setup)


@custom_op('noise_amd::clip_gradients', mutates_args=('gradients',))
def clip_gradients(gradients: List[Tensor], max_norm: float) -> Tensor:
    _backwards_only('clip_gradients')
    with torch.no_grad():
        return _clip.clip('clip_gradients', gradients, max_norm)


@clip_gradients.register_fake
def _clip_gradients_fake(gradients, max_norm):
    return gradients[0].new_empty((), dtype=torch.float32)


@custom_op('noise_amd::residual_norm', mutates_args=())
def residual_norm(x: Tensor, y: Optional[Tensor], x0: Optional[Tensor], scale: Optional[Tensor], x0_scale: Optional[Tensor],
                  gate: Optional[Tensor], y_weight: Optional[Tensor], weight: Optional[Tensor], norm_y: bool,
                  dtype: Optional[torch.dtype], eps: float) -> Tuple[Tensor, Tensor]:
    _backwards_only('residual_norm')
    return _residual.forward(x, y, x0, scale, x0_scale, gate, y_weight, weight, norm_y, dtype, eps)


@residual_norm.register_fake
def _residual_norm_fake(x, y, x0, scale, x0_scale, gate, y_weight, weight, norm_y, dtype, eps):
    return x.new_empty(x.shape), x.new_empty(x.shape, dtype=dtype or (x if y is None else y).dtype)


@custom_op('noise_amd::residual_norm_backward', mutates_args=())
def residual_norm_backward(dout: Optional[Tensor], dh: Optional[Tensor], x: Tensor, y: Optional[Tensor], x0: Optional[Tensor],
                           scale: Optional[Tensor], x0_scale: Optional[Tensor], gate: Optional[Tensor],
                           y_weight: Optional[Tensor], weight: Optional[Tensor], norm_y: bool, dtype: Optional[torch.dtype],
                           eps: float, needs: List[bool]) -> List[Tensor]:
    """The gradients that `needs` asks for, in its order (empty tensors in the others' places)"""
    _backwards_only('residual_norm_backward')
    grads = _residual.backward(dout, dh, x, y, x0, scale, x0_scale, gate, y_weight, weight, norm_y, dtype, eps, needs)
    return [x.new_empty(0) if g is None else g for g in grads]


@residual_norm_backward.register_fake
def _residual_norm_backward_fake(dout, dh, x, y, x0, scale, x0_scale, gate, y_weight, weight, norm_y, dtype, eps, needs):
    given = (x, y, x0, scale, x0_scale, gate, y_weight, weight)
    return [t.new_empty(t.shape) if n and t is not None else x.new_empty(0) for t, n in zip(given, needs)]


def _residual_norm_setup(ctx, inputs, output):
    *tensors, ctx.norm_y, ctx.dtype, ctx.eps = inputs
    ctx.save_for_backward(*tensors)
    ctx.set_materialize_grads(False)


def _residual_norm_backward(ctx, dout, dh):
    tensors, needs = ctx.saved_tensors, [bool(n) for n in ctx.needs_input_grad[:8]]
    grads = torch.ops.noise_amd.residual_norm_backward(dout, dh, *tensors, ctx.norm_y, ctx.dtype, ctx.eps, needs)
    return (*(g if n and t is not None else None for g, n, t in zip(grads, needs, tensors)), None, None, None)


residual_norm.register_autograd(_residual_norm_backward, setup_context=_residual_norm_setup)


@custom_op('noise_amd::linear_cross_entropy', mutates_args=())
def linear_cross_entropy(x: Tensor, weight: Tensor, targets: Tensor, vocab: int, softcap: Optional[float]) -> Tuple[Tensor, Tensor]:
    """The losses, and what their backward pass needs"""
    _backwards_only('linear_cross_entropy')
    return _vocab.forward(x, weight, targets, vocab, softcap, True)


@linear_cross_entropy.register_fake
def _linear_cross_entropy_fake(x, weight, targets, vocab, softcap):
    return x.new_empty(x.shape[:-1], dtype=torch.float32), x.new_empty(x.shape[:-1], dtype=torch.float32)


@custom_op('noise_amd::linear_cross_entropy_backward', mutates_args=())
def linear_cross_entropy_backward(dloss: Tensor, x: Tensor, weight: Tensor, targets: Tensor, lse: Tensor, vocab: int,
                                  softcap: Optional[float], need_x: bool, need_weight: bool) -> Tuple[Tensor, Tensor]:
    """dx and dweight (empty where not needed)"""
    _backwards_only('linear_cross_entropy_backward')
    grads = _vocab.gradients('linear_cross_entropy', x, weight, targets, dloss, lse, vocab, softcap, need_x, need_weight)[1:]
    return tuple(x.new_empty(0) if g is None else g for g in grads)


@linear_cross_entropy_backward.register_fake
def _linear_cross_entropy_backward_fake(dloss, x, weight, targets, lse, vocab, softcap, need_x, need_weight):
    return x.new_empty(x.shape if need_x else 0), weight.new_empty(weight.shape if need_weight else 0)


@custom_op('noise_amd::linear_cross_entropy_grad', mutates_args=())
def linear_cross_entropy_grad(x: Tensor, weight: Tensor, targets: Tensor, token_weight: Optional[Tensor], vocab: int,
                              softcap: Optional[float]) -> Tuple[Tensor, Tensor, Tensor]:
    _backwards_only('linear_cross_entropy_grad')
    return _vocab.gradients('linear_cross_entropy_grad', x, weight, targets, token_weight, None, vocab, softcap)


@linear_cross_entropy_grad.register_fake
def _linear_cross_entropy_grad_fake(x, weight, targets, token_weight, vocab, softcap):
    return x.new_empty(x.shape[:-1], dtype=torch.float32), x.new_empty(x.shape), weight.new_empty(weight.shape)


def _linear_cross_entropy_setup(ctx, inputs, output):
    x, weight, targets, *ctx.more = inputs
    ctx.mark_non_differentiable(output[1])
    ctx.save_for_backward(x, weight, targets, output[1])


def _linear_cross_entropy_backward(ctx, dloss, _):
    x, weight, targets, lse = ctx.saved_tensors
    needs = [bool(n) for n in ctx.needs_input_grad[:2]]
    grads = torch.ops.noise_amd.linear_cross_entropy_backward(dloss, x, weight, targets, lse, *ctx.more, *needs)
    return (*(g if n else None for g, n in zip(grads, needs)), None, None, None)


linear_cross_entropy.register_autograd(_linear_cross_entropy_backward, setup_context=_linear_cross_entropy_setup)
