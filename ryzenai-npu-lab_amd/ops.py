"""Per-operation entry points with the reference's names and call shapes.

Each function mirrors one @iron.jit entry point of the reference's
experiments/lfm25_*_kernel.py: the same positional tensors (inputs first,
preallocated outputs written in place, no return value) and the same
keyword-only compile-time integers. Tensors are torch tensors on the GPU
(BF16 as torch.bfloat16, ids as torch.int32), contiguous. Shape and dtype
errors raise ValueError before anything is launched; device errors raise
RuntimeError. Calls are stream-ordered on torch's current stream and return
without waiting; NPU-only knobs such as n_cores are validated and ignored.
"""

from __future__ import annotations

import functools
import struct

import torch

from . import _lib

HIDDEN, FFN, VOCAB = 1024, 2560, 65536
GAMMA_TILE = 4096  # the reference pads every norm weight to one 64x64 tile


if hasattr(torch._C, "_cuda_getCurrentRawStream") and hasattr(torch._C, "_cuda_getDevice"):
    def _stream() -> int:
        """The handle of torch's current stream (0.2 us; the Stream object
        that torch.cuda.current_stream() makes of it takes 2.8). Asked for
        after the arguments are known to be GPU tensors, so the device is
        initialized."""
        return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())
else:  # a torch without these private names
    def _stream() -> int:
        return torch.cuda.current_stream().cuda_stream


def _check(t: torch.Tensor, name: str, dtype: torch.dtype, numel: int | None = None) -> int:
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a torch tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a GPU tensor, got {t.device}")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if numel is not None and t.numel() != numel:
        raise ValueError(f"{name} must hold {numel} values, got {t.numel()}")
    return t.data_ptr()


def _bf(t, name, numel=None):
    return _check(t, name, torch.bfloat16, numel)


def _f32(t, name, numel=None):
    return _check(t, name, torch.float32, numel)


def _i32(t, name, numel=None):
    return _check(t, name, torch.int32, numel)


def _cores(n_cores: int) -> None:
    if n_cores not in (1, 2, 4):
        raise ValueError("n_cores must be 1, 2 or 4")


# ---------------------------------------------------------------- norms / GEMV

def rms_norm(input0, gamma0, output, *, N: int) -> None:
    """Reference: lfm25_rms_norm_kernel.py:16-53 (kernels/lfm25_rms_norm.cc)."""
    if not 1 <= N <= 65536:
        raise ValueError("N must be in [1, 65536]")
    _lib.call("lfm25_rms_norm", _bf(input0, "input0", N), _bf(gamma0, "gamma0", N),
              _bf(output, "output", N), N, _stream())


def bf16_bf16_gemv(weights, activation, output, *, M: int, K: int, n_cores: int = 4) -> None:
    """Reference: lfm25_bf16_gemv_kernel.py:18-114."""
    _cores(n_cores)
    if M < 1 or K < 8 or K % 8:
        raise ValueError("Needs M >= 1 and K divisible by 8")
    _lib.call("lfm25_bf16_bf16_gemv", _bf(weights, "weights", M * K),
              _bf(activation, "activation", K), _bf(output, "output", M), M, K, _stream())


def bf16_f32_gemv(weights, activation, output, *, M: int, K: int, n_cores: int = 4) -> None:
    """Reference: lfm25_gemv_kernel.py:21-109 (FP32 output)."""
    _cores(n_cores)
    if M < 1 or K < 8 or K % 8:
        raise ValueError("Needs M >= 1 and K divisible by 8")
    _lib.call("lfm25_bf16_f32_gemv", _bf(weights, "weights", M * K),
              _bf(activation, "activation", K), _f32(output, "output", M), M, K, _stream())


def norm_bf16_gemv(hidden, packed_gamma_and_weight, output, *, M: int, K: int) -> None:
    """Reference: lfm25_norm_gemv_kernel.py:18-122; packed = [gamma | pad to
    4096 | W row-major M x K] (006_lfm25_npu_norm_gemv.py:26-28)."""
    if K != 1024 or M < 1:
        raise ValueError("Needs K=1024 and M >= 1")
    _lib.call("lfm25_norm_bf16_gemv", _bf(hidden, "hidden", K),
              _bf(packed_gamma_and_weight, "packed_gamma_and_weight", GAMMA_TILE + M * K),
              _bf(output, "output", M), M, K, _stream())


def w8_gemv(weights, scales, activation, output, *, M: int, K: int, group: int) -> None:
    """INT8-weight GEMV in the formats of experiments/014_int8_lfm25.py:76-113
    (w8g32 / w8g64: group 32 / 64, FP32 scales [M, K / group]; w8c: group 0,
    FP32 scales [M]); weights int8 [M, K] as weights.quantize_w8 makes them."""
    if M < 1 or K < 64 or K > 4096 or K % 64:
        raise ValueError("Needs M >= 1 and K a multiple of 64 in [64, 4096]")
    if group not in (0, 32, 64):
        raise ValueError("group must be 0, 32 or 64")
    _lib.call("lfm25_w8_gemv", _check(weights, "weights", torch.int8, M * K),
              _f32(scales, "scales", M * (K // group if group else 1)),
              _bf(activation, "activation", K), _bf(output, "output", M), M, K, group, _stream())


def f32_to_bf16(input0, output, *, N: int) -> None:
    """Reference: lfm25_cast_kernel.py:16-45."""
    if N < 1:
        raise ValueError("N must be positive")
    _lib.call("lfm25_f32_to_bf16", _f32(input0, "input0", N), _bf(output, "output", N), N,
              _stream())


def bf16_add(left, right, output, *, N: int) -> None:
    """Reference: lfm25_add_kernel.py:16-53."""
    if N < 1:
        raise ValueError("N must be positive")
    _lib.call("lfm25_bf16_add", _bf(left, "left", N), _bf(right, "right", N),
              _bf(output, "output", N), N, _stream())


def silu_gate(w1, w3, output, *, N: int) -> None:
    """Reference: lfm25_silu_gate_kernel.py:16-51."""
    if N < 1:
        raise ValueError("N must be positive")
    _lib.call("lfm25_silu_gate", _bf(w1, "w1", N), _bf(w3, "w3", N), _bf(output, "output", N), N,
              _stream())


# ---------------------------------------------------------------- conv

def conv_gate(projection_and_weight, state, output, next_state) -> None:
    """Reference: lfm25_conv_gate_kernel.py:16-73; projection_and_weight =
    [B | C | x | w (1024 x 3)], state/next_state the HF [1024 x 3] state."""
    _lib.call("lfm25_conv_gate", _bf(projection_and_weight, "projection_and_weight", 6 * HIDDEN),
              _bf(state, "state", 3 * HIDDEN), _bf(output, "output", HIDDEN),
              _bf(next_state, "next_state", 3 * HIDDEN), _stream())


def conv_gate_packed_state(projection, state_and_weight, output, next_state_and_weight) -> None:
    """Reference: lfm25_conv_gate_packed_state_kernel.py:16-63."""
    _lib.call("lfm25_conv_gate_packed_state", _bf(projection, "projection", 3 * HIDDEN),
              _bf(state_and_weight, "state_and_weight", 6 * HIDDEN),
              _bf(output, "output", HIDDEN),
              _bf(next_state_and_weight, "next_state_and_weight", 6 * HIDDEN), _stream())


# [operator gamma tile | in_proj | out_proj | ffn gamma tile | w1 | w3 | w2]
_CONV_LAYER = 2 * GAMMA_TILE + (3 * HIDDEN + HIDDEN + 2 * FFN) * HIDDEN + HIDDEN * FFN


def _layer_workspace(device) -> torch.Tensor:
    """Scratch memory for one call of the layer programs (so concurrent calls
    never share one; the caching allocator hands the same memory out again)."""
    return torch.empty(_lib.load().lfm25_layer_workspace_bytes(), dtype=torch.uint8, device=device)


def recurrent_block(packed_hidden_and_state, packed_weights, next_state_and_weight,
                    block_output) -> None:
    """One conv decoder layer (lfm25_recurrent_block).
    Reference: lfm25_single_program_block_kernel.py:32-284.
    packed_hidden_and_state = [hidden (1024) | pad to 6144 | state (1024 x 3) |
    conv w (1024 x 3)]; packed_weights = [operator gamma tile | in_proj |
    out_proj | ffn gamma tile | w1 | w3 | w2]; next_state_and_weight =
    [next state (1024 x 3) | conv w (1024 x 3)]."""
    hp = _bf(packed_hidden_and_state, "packed_hidden_and_state", 2 * 6144)
    wp = _bf(packed_weights, "packed_weights", _CONV_LAYER)
    nxt = _bf(next_state_and_weight, "next_state_and_weight", 6144)
    out = _bf(block_output, "block_output", HIDDEN)
    ws = _layer_workspace(block_output.device)
    _lib.call("lfm25_recurrent_block", hp, hp + 2 * 6144, hp + 2 * (6144 + 3 * HIDDEN), wp, nxt, out, ws.data_ptr(),
              _stream())


# ---------------------------------------------------------------- attention

_QKV = HIDDEN + 2 * 512  # 2048


def attention_prefix(hidden, packed_weights, qkv_output, *, include_hidden: bool = False) -> None:
    """Operator norm, Q/K/V, per-head QK norm and RoPE.
    Reference: lfm25_attention_prefix_kernel.py:22-140; packed_weights =
    [gamma tile | q | k | v | aux tile = q_gamma (64) | k_gamma (64) | cos (64) |
    sin (64)]."""
    h = _bf(hidden, "hidden", HIDDEN)
    w = _bf(packed_weights, "packed_weights", 2 * GAMMA_TILE + _QKV * HIDDEN)
    out = _bf(qkv_output, "qkv_output", _QKV + (HIDDEN if include_hidden else 0))
    _lib.call("lfm25_attention_prefix", h, w, w + 2 * (GAMMA_TILE + _QKV * HIDDEN), out, 1 if include_hidden else 0,
              _stream())


def _past_length(cache, name: str) -> int:
    per = 2 * 8 * 64
    if cache.numel() % per:
        raise ValueError(f"{name} must hold 8 heads x 2 x past_length x 64 values")
    return cache.numel() // per


def attention_context(qkv, past_cache, context) -> None:
    """Reference: lfm25_attention_context_kernel.py:20-72 (past length taken
    from the cache size: 8 heads x [keys P x 64 | values P x 64])."""
    past = _past_length(past_cache, "past_cache")
    _lib.call("lfm25_attention_context", _bf(qkv, "qkv", _QKV), _bf(past_cache, "past_cache"),
              _bf(context, "context", HIDDEN), past, _stream())


def append_attention_cache(qkv, prior_cache, next_cache) -> None:
    """Reference: lfm25_attention_append_cache_kernel.py:20 (prior length P from
    prior_cache; next_cache holds P + 1 positions)."""
    past = _past_length(prior_cache, "prior_cache")
    _lib.call("lfm25_attention_append_cache", _bf(qkv, "qkv"), _bf(prior_cache, "prior_cache"),
              _bf(next_cache, "next_cache", 2 * 8 * (past + 1) * 64), past, _stream())


def attention_context_cache(qkv_and_hidden, past_cache, packed_tail_input, next_cache, *,
                            past_length: int = 21) -> None:
    """Context, KV append and tail-input packing in one call.
    Reference: lfm25_attention_context_cache_kernel.py:16-106;
    packed_tail_input = [hidden (1024) | context (1024)]."""
    if not 1 <= past_length < 4096:
        raise ValueError("past_length must be in [1, 4096)")
    qkv = _bf(qkv_and_hidden, "qkv_and_hidden", _QKV + HIDDEN)
    past = _bf(past_cache, "past_cache", 2 * 8 * past_length * 64)
    tail = _bf(packed_tail_input, "packed_tail_input", 2 * HIDDEN)
    nxt = _bf(next_cache, "next_cache", 2 * 8 * (past_length + 1) * 64)
    if (qkv | nxt) & 15:  # the one-pass form moves whole 16-byte pieces
        attention_context(qkv_and_hidden[:_QKV], past_cache, packed_tail_input[HIDDEN:])
        append_attention_cache(qkv_and_hidden[:_QKV], past_cache, next_cache)
        packed_tail_input[:HIDDEN].copy_(qkv_and_hidden[_QKV:])
        return
    ws = _layer_workspace(next_cache.device)
    _lib.call("lfm25_attention_context_cache", qkv, past, tail, nxt, past_length, ws.data_ptr(), _stream())


def attention_tail(packed_hidden_and_context, packed_weights, block_output) -> None:
    """o_proj + residual + SwiGLU MLP + residual.
    Reference: lfm25_attention_tail_kernel.py:29-208; packed_weights = [o |
    ffn gamma tile | w1 | w3 | w2]."""
    x = _bf(packed_hidden_and_context, "packed_hidden_and_context", 2 * HIDDEN)
    w = _bf(packed_weights, "packed_weights", HIDDEN * HIDDEN + GAMMA_TILE + 3 * FFN * HIDDEN)
    out = _bf(block_output, "block_output", HIDDEN)
    ws = _layer_workspace(block_output.device)
    _lib.call("lfm25_attention_tail", x, w, out, ws.data_ptr(), _stream())


# ---------------------------------------------------------------- head / embedding

def _workspace(count: int, device) -> torch.Tensor:
    n = int(_lib.load().lfm25_argmax_workspace_bytes(count))
    return torch.empty(n, dtype=torch.uint8, device=device)


def vocab_argmax(logits, token_id) -> None:
    """First index of the maximum BF16 logit. Reference: lfm25_argmax_kernel.py:18-68."""
    n = logits.numel()
    ws = _workspace(n, logits.device)
    _lib.call("lfm25_argmax", _bf(logits, "logits"), n, _i32(token_id, "token_id", 1),
              ws.data_ptr(), _stream())


def fused_vocab(hidden, packed_gamma_and_embedding, next_embedding, token_id, *,
                logits=None) -> None:
    """Final norm, tied head, argmax and the winning embedding row.
    Reference: lfm25_fused_vocab_kernel.py:22-110; packed = [gamma (1024) |
    E (vocab x 1024)] (vocab = 65536 in the reference; any multiple of 4 here)."""
    total = packed_gamma_and_embedding.numel()
    if total < HIDDEN or (total - HIDDEN) % HIDDEN:
        raise ValueError("packed_gamma_and_embedding must be [gamma | E (vocab x 1024)]")
    vocab = (total - HIDDEN) // HIDDEN
    if vocab < 4 or vocab % 4:
        raise ValueError("vocab must be a positive multiple of 4")
    ws = _workspace(vocab, hidden.device)
    lp = 0 if logits is None else _bf(logits, "logits", vocab)
    _lib.call("lfm25_fused_vocab", _bf(hidden, "hidden", HIDDEN),
              _bf(packed_gamma_and_embedding, "packed_gamma_and_embedding"),
              _bf(next_embedding, "next_embedding", HIDDEN), _i32(token_id, "token_id", 1), lp,
              vocab, ws.data_ptr(), _stream())


def embedding_dma_dynamic(table, embedding, token_id) -> None:
    """Reference: lfm25_embedding_dynamic_kernel.py:22-68 (id read on device)."""
    if table.dim() != 2 or table.shape[1] != HIDDEN:
        raise ValueError("table must be [vocab, 1024]")
    _lib.call("lfm25_embedding_gather", _bf(table, "table"), _i32(token_id, "token_id", 1),
              _bf(embedding, "embedding", HIDDEN), table.shape[0], 0, _stream())


def embedding_dma(table, embedding, *, token_id: int) -> None:
    """Reference: lfm25_embedding_dma_kernel.py:11-39 (id fixed at call time)."""
    if table.dim() != 2 or table.shape[1] != HIDDEN:
        raise ValueError("table must be [vocab, 1024]")
    if not 0 <= token_id < table.shape[0]:
        raise ValueError("Token ID outside vocabulary")
    tid = torch.tensor([token_id], dtype=torch.int32, device=table.device)
    embedding_dma_dynamic(table, embedding, tid)


def embedding_pair_dynamic(table, pair, token_ids) -> None:
    """Two embedding rows, ids read on the device: pair = [table[ids[0]] |
    table[ids[1]]]. Reference: lfm25_prefill_pair_embedding_kernel.py:18."""
    if table.dim() != 2 or table.shape[1] != HIDDEN:
        raise ValueError("table must be [vocab, 1024]")
    _bf(pair, "pair", 2 * HIDDEN)
    _i32(token_ids, "token_ids", 2)
    for i in range(2):
        _lib.call("lfm25_embedding_gather", table.data_ptr(), token_ids[i:i + 1].data_ptr(),
                  pair[i * HIDDEN:(i + 1) * HIDDEN].data_ptr(), table.shape[0], 0, _stream())


# ---------------------------------------------------------------- packing programs

def pack_block_input(hidden, state_and_weight, packed) -> None:
    """packed = [hidden | zeros to 6144 | state_and_weight (6144)].
    Reference: lfm25_pack_block_input_kernel.py:17 (kernels/lfm25_pack_block_input.cc)."""
    _lib.call("lfm25_pack_block_input", _bf(hidden, "hidden", HIDDEN),
              _bf(state_and_weight, "state_and_weight", 6144), _bf(packed, "packed", 12288), _stream())


def pack_conv(projection, weight, packed) -> None:
    """packed = [projection (3072) | weight (3072)].
    Reference: lfm25_pack_conv_kernel.py:17 (kernels/lfm25_pack_conv.cc)."""
    _lib.call("lfm25_pack_conv", _bf(projection, "projection", 3 * HIDDEN), _bf(weight, "weight", 3 * HIDDEN),
              _bf(packed, "packed", 6 * HIDDEN), _stream())


def pack_attention_tail(hidden, context, packed) -> None:
    """packed = [hidden | context].
    Reference: lfm25_pack_attention_tail_kernel.py:17 (kernels/lfm25_pack_attention_tail.cc)."""
    _lib.call("lfm25_pack_attention_tail", _bf(hidden, "hidden", HIDDEN), _bf(context, "context", HIDDEN),
              _bf(packed, "packed", 2 * HIDDEN), _stream())


def concat_hidden_pair(first, second, pair) -> None:
    """pair = [first | second]. Reference: lfm25_prefill_pair_data_kernel.py:11."""
    _lib.call("lfm25_concat_hidden_pair", _bf(first, "first", HIDDEN), _bf(second, "second", HIDDEN),
              _bf(pair, "pair", 2 * HIDDEN), _stream())


def split_hidden_pair(pair, first, second) -> None:
    """first, second = pair. Reference: lfm25_prefill_pair_data_kernel.py:42."""
    _lib.call("lfm25_split_hidden_pair", _bf(pair, "pair", 2 * HIDDEN), _bf(first, "first", HIDDEN),
              _bf(second, "second", HIDDEN), _stream())


def pack_recurrent_pair(pair, state, packed) -> None:
    """packed = [first | zeros to 6144 | second | zeros to 12288 | state (6144)].
    Reference: lfm25_prefill_pair_data_kernel.py:73."""
    _lib.call("lfm25_pack_recurrent_pair", _bf(pair, "pair", 2 * HIDDEN), _bf(state, "state", 6144),
              _bf(packed, "packed", 18432), _stream())


# ---------------------------------------------------------------- more layer programs

def norm_proj_conv(packed_hidden_and_state, packed_gamma_and_projection_weight, gate_output,
                   next_state_and_weight) -> None:
    """Operator norm, in_proj and the gated conv of a conv layer.
    Reference: lfm25_norm_proj_conv_kernel.py:24-148; packed_hidden_and_state =
    [hidden | pad to 6144 | state (1024 x 3) | conv w (1024 x 3)];
    packed_gamma_and_projection_weight = [gamma tile | in_proj (3072 x 1024)]."""
    _bf(packed_hidden_and_state, "packed_hidden_and_state", 2 * 6144)
    _bf(packed_gamma_and_projection_weight, "packed_gamma_and_projection_weight", GAMMA_TILE + 3 * HIDDEN * HIDDEN)
    _bf(gate_output, "gate_output", HIDDEN)
    _bf(next_state_and_weight, "next_state_and_weight", 6144)
    proj = torch.empty(3 * HIDDEN, dtype=torch.bfloat16, device=gate_output.device)
    norm_bf16_gemv(packed_hidden_and_state[:HIDDEN], packed_gamma_and_projection_weight, proj,
                   M=3 * HIDDEN, K=HIDDEN)
    conv_gate_packed_state(proj, packed_hidden_and_state[6144:], gate_output, next_state_and_weight)


def _pair_layer(hiddens, state_in, conv_w, packed_weights, next_state_and_weight, block_output) -> None:
    """Two consecutive positions through one conv layer: the second starts
    from the state the first left (lfm25_recurrent_block twice, in place)."""
    wp = _bf(packed_weights, "packed_weights", _CONV_LAYER)
    nxt = _bf(next_state_and_weight, "next_state_and_weight", 6144)
    out = _bf(block_output, "block_output", 2 * HIDDEN)
    ws = _layer_workspace(block_output.device)
    for i, h in enumerate(hiddens):
        _lib.call("lfm25_recurrent_block", h.data_ptr(), state_in.data_ptr() if i == 0 else nxt, conv_w.data_ptr(), wp,
                  nxt, out + 2 * i * HIDDEN, ws.data_ptr(), _stream())


def recurrent_pair_block(packed_hidden_and_state, packed_weights, next_state_and_weight, block_output) -> None:
    """Two prompt positions through one conv layer. Reference:
    lfm25_prefill_pair_block_kernel.py:33; packed_hidden_and_state = [first |
    pad to 6144 | second | pad to 12288 | state (1024 x 3) | conv w (1024 x 3)]
    (pack_recurrent_pair); packed_weights as recurrent_block; block_output =
    [first | second]."""
    _bf(packed_hidden_and_state, "packed_hidden_and_state", 3 * 6144)
    p = packed_hidden_and_state
    _pair_layer([p[:HIDDEN], p[6144:6144 + HIDDEN]], p[12288:12288 + 3 * HIDDEN], p[12288 + 3 * HIDDEN:],
                packed_weights, next_state_and_weight, block_output)


def recurrent_pair_direct(hidden_pair, prior_state_and_weight, packed_weights, next_state_and_weight,
                          block_output) -> None:
    """recurrent_pair_block with the pair and the state in separate buffers.
    Reference: lfm25_prefill_pair_direct_kernel.py:33."""
    _bf(hidden_pair, "hidden_pair", 2 * HIDDEN)
    _bf(prior_state_and_weight, "prior_state_and_weight", 6144)
    _pair_layer([hidden_pair[:HIDDEN], hidden_pair[HIDDEN:]], prior_state_and_weight[:3 * HIDDEN],
                prior_state_and_weight[3 * HIDDEN:], packed_weights, next_state_and_weight, block_output)


def attention_prefix_pair(hidden_pair, packed_weights_and_aux0, aux1, qkv_pair) -> None:
    """attention_prefix of two positions: qkv_pair = [q|k|v|hidden of the first
    (3072) | the same of the second]; aux0 (the first position's QK-norm and
    RoPE tile) ends packed_weights_and_aux0, aux1 is the second's.
    Reference: lfm25_prefill_pair_attention_prefix_kernel.py:23."""
    h = _bf(hidden_pair, "hidden_pair", 2 * HIDDEN)
    second = _bf(aux1, "aux1", GAMMA_TILE)
    out = _bf(qkv_pair, "qkv_pair", 2 * (_QKV + HIDDEN))
    w = _bf(packed_weights_and_aux0, "packed_weights_and_aux0", 2 * GAMMA_TILE + _QKV * HIDDEN)
    for i, aux in enumerate((w + 2 * (GAMMA_TILE + _QKV * HIDDEN), second)):
        _lib.call("lfm25_attention_prefix", h + 2 * i * HIDDEN, w, aux, out + 2 * i * (_QKV + HIDDEN), 1, _stream())


def attention_tail_pair(packed_hidden_and_context, packed_weights, block_output) -> None:
    """attention_tail of two positions: [hidden | context] of each in turn ->
    block_output = [first | second]. Reference:
    lfm25_prefill_pair_attention_tail_kernel.py:30."""
    _bf(packed_hidden_and_context, "packed_hidden_and_context", 4 * HIDDEN)
    _bf(block_output, "block_output", 2 * HIDDEN)
    for i in range(2):
        attention_tail(packed_hidden_and_context[2 * i * HIDDEN:2 * (i + 1) * HIDDEN], packed_weights,
                       block_output[i * HIDDEN:(i + 1) * HIDDEN])


# ---------------------------------------------------------------- headered KV caches

def _head_elems(capacity: int) -> int:
    return 2 + 2 * capacity * 64


def _attention_fixed(qkv_and_hidden, past_cache, packed_tail_input, next_cache, capacity: int,
                     blocks: int = 1) -> None:
    n = blocks * 8 * _head_elems(capacity)
    _bf(qkv_and_hidden, "qkv_and_hidden", _QKV + HIDDEN)
    _bf(packed_tail_input, "packed_tail_input", 2 * HIDDEN)
    _bf(next_cache, "next_cache", n)
    past = 0 if past_cache is None else _bf(past_cache, "past_cache", n)
    # The kernel reports a full or malformed block in bit 0 of a status word
    # and then leaves packed_tail_input and next_cache unwritten.
    status = torch.zeros(1, dtype=torch.int32, device=qkv_and_hidden.device)
    _lib.call("lfm25_attention_fixed", qkv_and_hidden.data_ptr(), past, packed_tail_input.data_ptr(),
              next_cache.data_ptr(), capacity, blocks, status.data_ptr(), _stream())
    if int(status.item()) & 1:
        raise ValueError(f"attention: a headered KV cache block (capacity {capacity}) is full or holds "
                         "a length outside [0, capacity); nothing was written")


def attention_first_context(qkv_and_hidden, packed_tail_input, first_cache) -> None:
    """Position 0: context = each KV head's value; first_cache = per head [k | v].
    Reference: lfm25_attention_first_context_kernel.py:16-17."""
    _lib.call("lfm25_attention_first_context", _bf(qkv_and_hidden, "qkv_and_hidden", _QKV + HIDDEN),
              _bf(packed_tail_input, "packed_tail_input", 2 * HIDDEN), _bf(first_cache, "first_cache", HIDDEN),
              _stream())


def attention_first_fixed(qkv_and_hidden, packed_tail_input, first_cache) -> None:
    """Position 0 into a capacity-32 headered cache.
    Reference: lfm25_attention_fixed_cache_kernel.py:30-31."""
    _attention_fixed(qkv_and_hidden, None, packed_tail_input, first_cache, 32)


def attention_context_fixed(qkv_and_hidden, past_cache, packed_tail_input, next_cache) -> None:
    """Attention and append over a capacity-32 headered cache.
    Reference: lfm25_attention_fixed_cache_kernel.py:81-82."""
    _attention_fixed(qkv_and_hidden, past_cache, packed_tail_input, next_cache, 32)


def attention_first_fixed64(qkv_and_hidden, packed_tail_input, first_cache) -> None:
    """Position 0 into a capacity-64 headered cache.
    Reference: lfm25_attention_fixed64_cache_kernel.py:31."""
    _attention_fixed(qkv_and_hidden, None, packed_tail_input, first_cache, 64)


def attention_context_fixed64(qkv_and_hidden, past_cache, packed_tail_input, next_cache) -> None:
    """Attention and append over a capacity-64 headered cache.
    Reference: lfm25_attention_fixed64_cache_kernel.py:82."""
    _attention_fixed(qkv_and_hidden, past_cache, packed_tail_input, next_cache, 64)


def attention_context_chunked(qkv_and_hidden, past_cache, packed_tail_input, next_cache, *,
                              block_count: int = 1) -> None:
    """Attention and append over `block_count` capacity-64 blocks (positions
    in block order, the new one appended to the last block).
    Reference: lfm25_attention_chunked_cache_kernel.py:22-24."""
    if not 1 <= block_count <= 64:
        raise ValueError("block_count must be in [1, 64]")
    _attention_fixed(qkv_and_hidden, past_cache, packed_tail_input, next_cache, 64, block_count)


def attention_pair_context_fixed64(qkv_pair, past_cache, tail_pair, next_cache) -> None:
    """Two causal positions over a capacity-64 headered cache: the second
    attends to the first. tail_pair = [hidden | context of the first | the
    same of the second]. Reference: lfm25_prefill_pair_attention_context_kernel.py:22."""
    _bf(qkv_pair, "qkv_pair", 2 * (_QKV + HIDDEN))
    _bf(tail_pair, "tail_pair", 4 * HIDDEN)
    step = _QKV + HIDDEN
    _attention_fixed(qkv_pair[:step], past_cache, tail_pair[:2 * HIDDEN], next_cache, 64)
    _attention_fixed(qkv_pair[step:], next_cache, tail_pair[2 * HIDDEN:], next_cache, 64)


# ---------------------------------------------------------------- vocabulary, matmul

def fused_vocab_4core(hidden, packed_gamma_and_embedding, next_embedding, token_id) -> None:
    """fused_vocab over the full 65,536-row vocabulary (the NPU's four-core
    shard split has no counterpart: the GPU scans every row in one launch).
    Reference: lfm25_fused_vocab_4core_kernel.py:24-26."""
    if packed_gamma_and_embedding.numel() != HIDDEN + VOCAB * HIDDEN:
        raise ValueError("packed_gamma_and_embedding must be [gamma | E (65536 x 1024)]")
    fused_vocab(hidden, packed_gamma_and_embedding, next_embedding, token_id)


def bf16_f32_matmul(input0, input1, output, *, M: int, K: int, N: int, n_cores: int = 1,
                    reuse_weights: bool = False) -> None:
    """output[M x N] (FP32) = input0[M x K] . input1[K x N] (BF16, row-major).
    Reference: lfm25_matmul_kernel.py:16-27 (same shape checks)."""
    if M < 16 or M % 16 or K % 64 or n_cores not in (1, 2, 4) or N % (64 * n_cores):
        raise ValueError("Needs M%16=0, K%64=0, N%(64*n_cores)=0, cores in 1/2/4")
    if reuse_weights and M != 48:
        raise ValueError("Weight reuse probe requires M=48")
    _lib.call("lfm25_bf16_f32_matmul", _bf(input0, "input0", M * K), _bf(input1, "input1", K * N),
              _f32(output, "output", M * N), M, K, N, _stream())


# ---------------------------------------------------------------- paged 8-bit KV cache
#
# A pool of pages of `page` positions in int8 or FP8 (e4m3), one FP32 scale
# per page and KV head; block tables give each request's pages. A pass is
# kv8_plan, then per layer kv8_append and kv8_attention (lfm25_kv8_* in
# include/lfm25_hip.h has the definitions). Nothing here waits for the GPU,
# and all of it may be captured into a graph.
#
# These calls are short, so their checks are one expression each (a tensor's
# attribute costs 0.07 us, a call 0.1), and the arguments go over as one packed
# structure (0.5 us; 24 separate ones take ctypes 2.0): 12.5 -> 6 us a call,
# of which 4 are the launch.
# Where the expression is false, the checks one by one name what is wrong.

KV8_LENGTH, KV8_TABLE, KV8_POOL, KV8_ROWS = 1, 2, 4, 8  # kv8_plan's status
KV8_BAD_PAGE, KV8_BAD_ROWS = 1, 2                       # kv8_attention's status bits
_KV8_FORMATS = {torch.int8: 0, torch.float8_e4m3fn: 1}
_KV8_PAGES = frozenset((16, 32, 64, 128, 256))
_KV8_MAX_REQUESTS = 4096
_BF16, _F32, _INT32, _INT64 = torch.bfloat16, torch.float32, torch.int32, torch.int64

_PLAN = struct.Struct("@9P5i")
_PLAN_PAGES = struct.Struct("@2P")
_APPEND = struct.Struct("@7P2q6i")
_ATTEND = struct.Struct("@11Pq11if")


if hasattr(torch._C, "_cuda_getCurrentRawStream") and hasattr(torch._C, "_cuda_getDevice"):
    _device, _stream_of = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
else:  # a torch without these private names
    _device = torch.cuda.current_device

    def _stream_of(device: int) -> int:
        return torch.cuda.current_stream(device).cuda_stream


def _here(*tensors) -> None:
    """All on the current device, whose stream the call goes to."""
    device = torch.cuda.current_device()
    for t in tensors:
        if t.get_device() != device:
            raise ValueError(f"tensors must be on the current device (cuda:{device}), got {t.device}")


def _kv8_rows(t, name: str, heads: int, dim: int, rows: int) -> None:
    """BF16 rows [rows, heads, dim], which may be apart."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a GPU tensor")
    if t.dtype != _BF16:
        raise ValueError(f"{name} must be {_BF16}, got {t.dtype}")
    if t.shape != (rows, heads, dim):
        raise ValueError(f"{name} must be [{rows}, {heads}, {dim}], got {list(t.shape)}")
    s = t.stride()
    if s[2] != 1 or (heads > 1 and s[1] != dim):
        raise ValueError(f"{name}: a row's heads must be contiguous")


def _kv8_cache(key_cache, value_cache, key_scales, value_scales):
    """(pages, kv_heads, page, dim) of a cache's four tensors."""
    if not isinstance(key_cache, torch.Tensor) or key_cache.dim() != 4:
        raise ValueError("key_cache must be [pages, kv_heads, page, dim]")
    if key_cache.dtype not in _KV8_FORMATS:
        raise ValueError(f"key_cache must be torch.int8 or torch.float8_e4m3fn, got {key_cache.dtype}")
    pages, kv, page, dim = key_cache.shape
    if page not in _KV8_PAGES or dim not in (64, 128):
        raise ValueError(f"pages must be of 16, 32, 64, 128 or 256 positions and dim 64 or 128, got {page} and {dim}")
    _check(key_cache, "key_cache", key_cache.dtype)
    _check(value_cache, "value_cache", key_cache.dtype)
    if value_cache.shape != (pages, kv, dim, page):
        raise ValueError(f"value_cache must be [{pages}, {kv}, {dim}, {page}], got {list(value_cache.shape)}")
    _f32(key_scales, "key_scales", pages * kv)
    _f32(value_scales, "value_scales", pages * kv)
    return pages, kv, page, dim


def _kv8_table(block_table, requests: int) -> None:
    _i32(block_table, "block_table")
    if block_table.dim() != 2 or block_table.shape[0] != requests or block_table.shape[1] < 1:
        raise ValueError(f"block_table must be [{requests}, width]")


def _kv8_requests(past) -> int:
    if isinstance(past, torch.Tensor) and not 1 <= past.numel() <= _KV8_MAX_REQUESTS:
        raise ValueError(f"past must hold 1 to {_KV8_MAX_REQUESTS} lengths")
    _i32(past, "past")
    return past.numel()


def _kv8_plan_check(past, counts, block_table, free_pages, cursor, row_starts, slots, next_cursor, status, page) -> None:
    if page not in _KV8_PAGES:
        raise ValueError("page must be 16, 32, 64, 128 or 256")
    n = _kv8_requests(past)
    _i32(counts, "counts", n)
    _kv8_table(block_table, n)
    _i32(free_pages, "free_pages")
    _check(cursor, "cursor", _INT64, 2)
    _i32(row_starts, "row_starts", n + 1)
    _i32(slots, "slots")
    _check(next_cursor, "next_cursor", _INT64, 2)
    _i32(status, "status", n)
    if free_pages.numel() < 1 or slots.numel() < 1:
        raise ValueError("free_pages and slots must not be empty")
    _here(past, counts, block_table, free_pages, cursor, row_starts, slots, next_cursor, status)


def _kv8_plan_pages(requests: int, **pages) -> bytes:
    for name, t in pages.items():
        if t is not None:
            _i32(t, name, requests)
            _here(t)
    return _PLAN_PAGES.pack(*(0 if t is None else t.data_ptr() for t in pages.values()))


def kv8_plan(past, counts, block_table, free_pages, cursor, row_starts, slots, next_cursor, status, *, page: int,
             shared=None, held=None) -> None:
    """Pages, row offsets and cache slots of a pass from the requests' lengths
    (lfm25_kv8_plan). past, counts: int32 [requests], positions held and new
    rows (counts[b] < 0 ends request b and gives its pages back). block_table:
    int32 [requests, width], extended in place. free_pages: int32 [ring], a
    ring of free page numbers, of which the entries cursor[0] .. cursor[1]
    (int64, counted on without end) are free. Written: row_starts int32
    [requests + 1], slots int32 [rows] (-1: a refused request's row, or behind
    the last), next_cursor int64 [2] (may be cursor), status int32 [requests]
    (0, or KV8_LENGTH / KV8_TABLE / KV8_POOL / KV8_ROWS).

    A page may be in several rows of the table, but is one request's own, which
    ends after the others that have it: shared, int32 [requests], says how many
    pages at its beginning are not a request's own. They are neither given
    back when it ends nor written to. Where lengths may go back (rejected
    drafts), held, int32 [requests], 0 at first and updated in place, keeps the
    pages in each row of the table; otherwise those behind a length that went
    back are lost (lfm25_kv8_plan_with)."""
    try:
        n, ring, rows, here = past.numel(), free_pages.numel(), slots.numel(), past.get_device()
        wide = block_table.shape
        fine = (page in _KV8_PAGES and 1 <= n <= _KV8_MAX_REQUESTS and ring > 0 and rows > 0 and len(wide) == 2
                and wide[0] == n and wide[1] > 0 and here >= 0
                and past.dtype is _INT32 and counts.dtype is _INT32 and block_table.dtype is _INT32
                and free_pages.dtype is _INT32 and row_starts.dtype is _INT32 and slots.dtype is _INT32
                and status.dtype is _INT32 and cursor.dtype is _INT64 and next_cursor.dtype is _INT64
                and counts.numel() == n and row_starts.numel() == n + 1 and status.numel() == n
                and cursor.numel() == 2 and next_cursor.numel() == 2
                and past.is_contiguous() and counts.is_contiguous() and block_table.is_contiguous()
                and free_pages.is_contiguous() and row_starts.is_contiguous() and slots.is_contiguous()
                and status.is_contiguous() and cursor.is_contiguous() and next_cursor.is_contiguous()
                and here == counts.get_device() == block_table.get_device() == free_pages.get_device()
                == row_starts.get_device() == slots.get_device() == status.get_device() == cursor.get_device()
                == next_cursor.get_device() and here == _device())
    except AttributeError:
        fine = False
    if not fine:
        _kv8_plan_check(past, counts, block_table, free_pages, cursor, row_starts, slots, next_cursor, status, page)
    call = _PLAN.pack(
        past.data_ptr(), counts.data_ptr(), block_table.data_ptr(), free_pages.data_ptr(), cursor.data_ptr(),
        row_starts.data_ptr(), slots.data_ptr(), next_cursor.data_ptr(), status.data_ptr(), n, wide[1], ring, rows, page)
    if shared is None and held is None:
        _lib.call("lfm25_kv8_plan", call, _stream_of(here))
    else:
        _lib.call("lfm25_kv8_plan_with", call, _kv8_plan_pages(n, shared=shared, held=held), _stream_of(here))


def _kv8_append_check(keys, values, slots, key_cache, value_cache, key_scales, value_scales) -> None:
    _, kv, _, dim = _kv8_cache(key_cache, value_cache, key_scales, value_scales)
    _i32(slots, "slots")
    _kv8_rows(keys, "keys", kv, dim, slots.numel())
    _kv8_rows(values, "values", kv, dim, slots.numel())
    _here(keys, values, slots, key_cache, value_cache, key_scales, value_scales)


def kv8_append(keys, values, slots, key_cache, value_cache, key_scales, value_scales) -> None:
    """New keys and values into the 8-bit cache (lfm25_kv8_append). keys,
    values: BF16 [rows, kv_heads, dim], rows may be strided (slices of a fused
    q | k | v product). slots: int32 [rows] as kv8_plan gives them (-1 leaves a
    row out). Written in place: key_cache [pages, kv_heads, page, dim] and
    value_cache [pages, kv_heads, dim, page] in torch.int8 or
    torch.float8_e4m3fn, key_scales and value_scales FP32 [pages, kv_heads]."""
    try:
        pages, kv, page, dim = key_cache.shape
        rows, here, code = slots.numel(), slots.get_device(), key_cache.dtype
        ks, vs = keys.stride(), values.stride()
        fine = (here >= 0 and code in _KV8_FORMATS and value_cache.dtype is code and page in _KV8_PAGES
                and (dim == 64 or dim == 128) and value_cache.shape == (pages, kv, dim, page)
                and keys.shape == values.shape == (rows, kv, dim) and ks[2] == vs[2] == 1
                and (kv == 1 or ks[1] == vs[1] == dim)
                and keys.dtype is _BF16 and values.dtype is _BF16 and slots.dtype is _INT32
                and key_scales.dtype is _F32 and value_scales.dtype is _F32
                and key_scales.numel() == value_scales.numel() == pages * kv
                and slots.is_contiguous() and key_cache.is_contiguous() and value_cache.is_contiguous()
                and key_scales.is_contiguous() and value_scales.is_contiguous()
                and here == keys.get_device() == values.get_device() == key_cache.get_device()
                == value_cache.get_device() == key_scales.get_device() == value_scales.get_device() and here == _device())
    except (AttributeError, ValueError, IndexError):
        fine = False
    if not fine:
        _kv8_append_check(keys, values, slots, key_cache, value_cache, key_scales, value_scales)
    if rows == 0:
        return
    _lib.call("lfm25_kv8_append", _APPEND.pack(
        keys.data_ptr(), values.data_ptr(), slots.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(),
        key_scales.data_ptr(), value_scales.data_ptr(), ks[0] if rows > 1 else kv * dim, vs[0] if rows > 1 else kv * dim,
        rows, pages, page, kv, dim, _KV8_FORMATS[code]), _stream_of(here))


@functools.lru_cache(maxsize=256)
def _kv8_workspace_bytes(*sizes: int) -> int:
    return int(_lib.load().lfm25_kv8_attention_workspace_bytes(*sizes))


def _kv8_attention_check(query, key_cache, value_cache, key_scales, value_scales, block_table, past, row_starts, output,
                         status, max_rows, scale) -> None:
    _, kv, _, dim = _kv8_cache(key_cache, value_cache, key_scales, value_scales)
    _bf(output, "output")
    if output.dim() != 3 or output.shape[2] != dim or output.shape[1] % kv or not 1 <= output.shape[1] // kv <= 16:
        raise ValueError(f"output must be [rows, heads, {dim}] with heads a multiple (1 to 16) of {kv}")
    _kv8_rows(query, "query", output.shape[1], dim, output.shape[0])
    n = _kv8_requests(past)
    _i32(row_starts, "row_starts", n + 1)
    _kv8_table(block_table, n)
    if max_rows < 1:
        raise ValueError("max_rows must be positive")
    if not 0.0 <= scale < float("inf"):
        raise ValueError("scale must be finite and not negative")
    tensors = [query, key_cache, value_cache, key_scales, value_scales, block_table, past, row_starts, output]
    if status is not None:
        _i32(status, "status", 1)
        tensors.append(status)
    _here(*tensors)


def kv8_attention(query, key_cache, value_cache, key_scales, value_scales, block_table, past, row_starts, output, *,
                  max_rows: int, scale: float | None = None, status=None) -> None:
    """Causal attention of a pass's rows over the 8-bit cache
    (lfm25_kv8_attention). query: BF16 [rows, heads, dim], rows may be strided;
    heads a multiple (up to 16) of the cache's kv_heads. block_table int32
    [requests, width], past int32 [requests], row_starts int32 [requests + 1]:
    row i of request b stands at position past[b] + i and sees the positions up
    to it, which kv8_append has written. max_rows: the most rows of one
    request. scale: of the scores, 1 / sqrt(dim) by default. Written: output
    BF16 [rows, heads, dim], contiguous; status (int32 [1], optional) gets bits
    KV8_BAD_PAGE / KV8_BAD_ROWS set."""
    try:
        pages, kv, page, dim = key_cache.shape
        rows, heads, width = output.shape
        n, here, code = past.numel(), past.get_device(), key_cache.dtype
        qs, table = query.stride(), block_table.shape
        if scale is None:
            scale = dim ** -0.5
        fine = (here >= 0 and width == dim and heads % kv == 0 and 1 <= heads // kv <= 16 and 1 <= n <= _KV8_MAX_REQUESTS
                and max_rows >= 1 and 0.0 <= scale < 3.4e38 and code in _KV8_FORMATS and value_cache.dtype is code
                and page in _KV8_PAGES and (dim == 64 or dim == 128) and value_cache.shape == (pages, kv, dim, page)
                and query.shape == output.shape and qs[2] == 1 and (heads == 1 or qs[1] == dim)
                and len(table) == 2 and table[0] == n and table[1] > 0
                and query.dtype is _BF16 and output.dtype is _BF16 and block_table.dtype is _INT32 and past.dtype is _INT32
                and row_starts.dtype is _INT32 and key_scales.dtype is _F32 and value_scales.dtype is _F32
                and row_starts.numel() == n + 1 and key_scales.numel() == value_scales.numel() == pages * kv
                and output.is_contiguous() and key_cache.is_contiguous() and value_cache.is_contiguous()
                and key_scales.is_contiguous() and value_scales.is_contiguous() and block_table.is_contiguous()
                and past.is_contiguous() and row_starts.is_contiguous()
                and here == query.get_device() == key_cache.get_device() == value_cache.get_device()
                == key_scales.get_device() == value_scales.get_device() == block_table.get_device()
                == row_starts.get_device() == output.get_device() and here == _device()
                and (status is None or (status.dtype is _INT32 and status.numel() == 1 and status.get_device() == here)))
    except (AttributeError, ValueError, IndexError, TypeError, ZeroDivisionError):
        fine = False
    if not fine:
        _kv8_attention_check(query, key_cache, value_cache, key_scales, value_scales, block_table, past, row_starts, output,
                             status, max_rows, 0.0 if scale is None else scale)
    if rows == 0:
        return
    if max_rows > rows:
        max_rows = rows
    need = _kv8_workspace_bytes(rows, heads, kv, dim, n, max_rows, table[1], page)
    # (the memory may go to another call of this stream once this one is queued)
    workspace = torch.empty(need, dtype=torch.uint8, device=output.device) if need else None
    _lib.call("lfm25_kv8_attention", _ATTEND.pack(
        query.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(), key_scales.data_ptr(), value_scales.data_ptr(),
        block_table.data_ptr(), past.data_ptr(), row_starts.data_ptr(), output.data_ptr(),
        0 if status is None else status.data_ptr(), workspace.data_ptr() if need else 0,
        qs[0] if rows > 1 else heads * dim, table[1], n, rows, heads, max_rows, pages, page, kv, dim,
        _KV8_FORMATS[code], 0, scale), _stream_of(here))
