"""LLaMA-style causal LM whose compute runs on the gfx950 HIP kernels.

Module tree, class names, attribute names, state_dict keys, constructor
signatures and the order of parameter construction follow the reference
(model/llama.py:14-335), so checkpoints, the ZeRO engines' flat layouts and the
seeded initial weights carry over.  The forward/backward math is the
reference's; it is computed by lzhip (RMSNorm, RoPE, fused QKV + flash
attention, fused gate/up + SwiGLU, GEMMs with the residual add in the
epilogue, embedding, cross entropy).  Tensors must live on a ROCm GPU; there is
no CPU compute path.
"""
from __future__ import annotations

import itertools
import numbers
import operator
import threading
from dataclasses import dataclass
from typing import Any, Callable, List, Optional, Sequence, Tuple, Union

import torch
import torch.nn as nn
from torch.utils.checkpoint import checkpoint as activation_checkpoint

from lzhip import functional as LF
from lzhip import ops
from lzhip.cache import CacheStep, DraftCache, DraftStep, KVCache, LayerCache

from .config import ModelConfig


def _next_token(logits: torch.Tensor, temperature: float, top_k: Optional[int]) -> torch.Tensor:
    """One token per row of [B, V] logits (see LlamaForCausalLM.generate)."""
    if temperature <= 0:
        return logits.argmax(dim=-1)
    scaled = _cut(logits / temperature, top_k)
    return torch.multinomial(torch.softmax(scaled, dim=-1), num_samples=1).squeeze(-1)


def _cut(logits: torch.Tensor, top_k: Optional[int]) -> torch.Tensor:
    """The rows' top_k largest logits, the others -inf."""
    if top_k is None:
        return logits
    kth = torch.topk(logits, min(top_k, logits.size(-1))).values[:, -1:]
    return logits.masked_fill(logits < kth, float("-inf"))


class _Tree:
    """Drafted tokens of one sequence: the root, and `widths[i]` children of
    each node of level i.  Nodes are numbered level by level."""

    def __init__(self, widths: Sequence[int]) -> None:
        self.widths = list(widths)
        self.levels, self.parents = [(0, 1)], [-1]
        for w in self.widths:
            lo, hi = self.levels[-1]
            self.parents += [p for p in range(lo, hi) for _ in range(w)]
            self.levels.append((hi, len(self.parents)))
        self.nodes = len(self.parents)

    def step_of(self, step: DraftStep, level: int) -> DraftStep:
        """The rows of a level, of a step that made room for all nodes."""
        lo, hi = self.levels[level]
        B, n = step.kv_len.numel(), hi - lo
        of = lambda t: t.view(B, self.nodes, *t.shape[1:])[:, lo:hi].reshape(B * n, *t.shape[1:]).contiguous()  # noqa: E731
        return step._replace(row_start=torch.arange(0, B * n + 1, n, dtype=torch.int32, device=step.kv_len.device),
                             kv_len=step.base + hi, rows=B * n, max_new=n, positions=of(step.positions), slots=of(step.slots),
                             mask=None if step.mask is None else of(step.mask))


def _require_choice(logits: torch.Tensor, t: int, temperature: float) -> None:
    """Refuses adjusted logits that leave a row no token t to choose (sampling
    from such a row would end the process).  Waits for the device."""
    top = logits.amax(-1)
    fine = top > float("-inf")  # not for NaN
    if temperature > 0:
        fine &= top < float("inf")
    if bool(fine.all()):
        return
    if bool(top.isnan().any()):
        why = "a row's logits hold NaN"
    elif bool((top == float("-inf")).any()):
        why = "token_mask or logit_bias allows a row no token"
    else:
        why = "a row's largest logit is infinite: it can be chosen (temperature 0) but not sampled"
    raise ValueError(f"token {t}: {why}")


class HipLinear(nn.Linear):
    """nn.Linear (same parameters, initialisation and state_dict) whose
    forward is the MFMA GEMM; bias is not supported (the model has none)."""

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        if self.bias is not None:
            raise NotImplementedError("HipLinear has no bias path")
        return LF.linear(x, self.weight, residual)


class HipLMHead(HipLinear):
    """The LM head (nn.Linear, tied to the embedding).  Called with labels it
    returns the shifted cross-entropy loss instead of the logits, through the
    fused LM-head + loss Function, which never holds the [B*S, V] logits."""

    fused_chunk_bytes = 1 << 30  # logits buffer of the fused loss

    def forward(self, x: torch.Tensor, labels: Optional[torch.Tensor] = None, clamp: bool = False) -> torch.Tensor:
        if labels is None:
            return super().forward(x)
        if self.bias is not None:
            raise NotImplementedError("the fused LM-head loss has no bias path")
        return LF.lm_head_cross_entropy(x, self.weight, labels, clamp, self.fused_chunk_bytes)


class HipEmbedding(nn.Embedding):
    """nn.Embedding (same parameters and initialisation) with the HIP gather."""

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        return LF.EmbeddingFn.apply(ids, self.weight)


class RMSNorm(nn.Module):
    def __init__(self, hidden_size: int, eps: float = 1e-6) -> None:
        super().__init__()
        self.weight = nn.Parameter(torch.ones(hidden_size))
        self.eps = eps

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return LF.rms_norm(x, self.weight, self.eps)

    def forward_with_residual(self, x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """(norm(x), x) for a pre-norm residual block; the residual gradient is
        added inside the norm's backward kernel."""
        return LF.rms_norm_with_residual(x, self.weight, self.eps)


def rotate_half(x: torch.Tensor) -> torch.Tensor:
    """cat(-x2, x1) over the last dimension (model/llama.py:25-28); a tensor
    helper kept for API compatibility, not used by the training path."""
    h = x.shape[-1] // 2
    return torch.cat((-x[..., h:], x[..., :h]), dim=-1)


def apply_rotary_pos_emb(
    q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor
) -> Tuple[torch.Tensor, torch.Tensor]:
    """q/k [..., S, hd] with tables [1, 1, S, hd] (model/llama.py:31-39)."""
    seq, hd = q.shape[-2], q.shape[-1]
    c2, s2 = cos.reshape(-1, hd)[:seq], sin.reshape(-1, hd)[:seq]
    return LF.RopeFn.apply(q, c2, s2), LF.RopeFn.apply(k, c2, s2)


_tables_lock = threading.Lock()  # of every module's rotary tables


class _Built:
    """The streams that may use tensors which the current one is building: the
    others wait for it once, and their work is waited for before the memory
    goes to another tensor.  A copy of a module copies its tensors, not this."""

    def __init__(self, device: torch.device) -> None:
        self.event = torch.cuda.current_stream(device).record_event()
        self.streams = {ops.stream_ptr(device)}

    def reach(self, device: torch.device, *tensors: torch.Tensor) -> None:
        if ops.stream_ptr(device) in self.streams:
            return
        stream = torch.cuda.current_stream(device)
        stream.wait_event(self.event)
        for t in tensors:
            t.record_stream(stream)
        self.streams.add(ops.stream_ptr(device))

    def __deepcopy__(self, memo) -> None:
        return None

    def __reduce__(self):
        return type(None), ()


class RotaryEmbedding(nn.Module):
    """cos/sin cache [1, 1, S, hd] in the activation dtype, rebuilt when the
    sequence grows or the device/dtype changes (model/llama.py:42-69); the
    table is computed by the lz_rope_table kernel from the inv_freq buffer.
    Like the reference's, that buffer follows Module.to(dtype), and the
    positions and angles are then formed in its dtype."""

    def __init__(self, dim: int, base: float = 500_000.0) -> None:
        super().__init__()
        self.dim = dim
        self.base = float(base)
        inv_freq = 1.0 / (base ** (torch.arange(0, dim, 2).float() / dim))
        self.register_buffer("inv_freq", inv_freq, persistent=False)
        self.max_seq_len_cached = 0
        self._captured = []  # tables that a captured call reads
        self._built: Optional[_Built] = None
        self.register_buffer("cos_cached", torch.empty(0), persistent=False)
        self.register_buffer("sin_cached", torch.empty(0), persistent=False)

    def _build_cache(self, seq_len: int, device: torch.device, dtype: torch.dtype) -> None:
        inv = self.inv_freq
        if inv.device != device:
            inv = inv.to(device)
        cos, sin = ops.rope_table(seq_len, self.dim, inv.contiguous(), dtype)
        self.cos_cached = cos[None, None]
        self.sin_cached = sin[None, None]
        self.max_seq_len_cached = seq_len

    def _tables(self, seq_len: int, device: torch.device, dtype: torch.dtype, block: int = 1
                ) -> Tuple[torch.Tensor, torch.Tensor]:
        """The cache, at least seq_len long, for the current stream.  Under
        capture: tables that the graph keeps an address of stay, whatever
        replaces them in the cache; what is built there (and by each replay) is
        the graph's alone, since it holds nothing before a replay."""
        with _tables_lock:
            cos, sin = self.cos_cached, self.sin_cached
            if seq_len <= self.max_seq_len_cached and cos.device == device and cos.dtype == dtype:
                if ops.capturing():
                    if not any(kept is cos for kept, _ in self._captured):
                        self._captured.append((cos, sin))
                elif self._built is not None:
                    self._built.reach(device, cos, sin)
                return cos, sin
            old = cos, sin, self.max_seq_len_cached
            self._build_cache(seq_len=-(-seq_len // block) * block, device=device, dtype=dtype)
            cos, sin = self.cos_cached, self.sin_cached
            if ops.capturing():
                self.cos_cached, self.sin_cached, self.max_seq_len_cached = old
            else:
                self._built = _Built(device) if device.type == "cuda" else None
            return cos, sin

    def forward(self, seq_len: int, device: torch.device, dtype: torch.dtype) -> Tuple[torch.Tensor, torch.Tensor]:
        cos, sin = self._tables(seq_len, device, dtype)
        return cos[:, :, :seq_len, :], sin[:, :, :seq_len, :]

    def tables(self, seq_len: int, device: torch.device, dtype: torch.dtype, block: int = 1
               ) -> Tuple[torch.Tensor, torch.Tensor]:
        """[S, hd] views of the cache for the fused kernels (of what forward()
        returns where that is replaced).  A position's rotation does not depend
        on the table's length: with block > 1 the cache grows to multiples of
        it, so that a growing sequence rarely rebuilds it."""
        forward = self.forward
        if getattr(forward, "__func__", None) is not RotaryEmbedding.forward:
            cos, sin = forward(seq_len, device, dtype)
            return cos.reshape(-1, self.dim), sin.reshape(-1, self.dim)
        cos, sin = self._tables(seq_len, device, dtype, block)
        return cos.view(-1, self.dim).narrow(0, 0, seq_len), sin.view(-1, self.dim).narrow(0, 0, seq_len)


class GroupedQueryAttention(nn.Module):
    def __init__(self, cfg: ModelConfig) -> None:
        super().__init__()
        self.n_heads = cfg.n_heads
        self.n_kv_heads = cfg.n_kv_heads
        self.head_dim = cfg.head_dim
        self.dropout = cfg.dropout
        self.scale = self.head_dim**-0.5

        self.q_proj = HipLinear(cfg.dim, cfg.n_heads * self.head_dim, bias=False)
        self.k_proj = HipLinear(cfg.dim, cfg.n_kv_heads * self.head_dim, bias=False)
        self.v_proj = HipLinear(cfg.dim, cfg.n_kv_heads * self.head_dim, bias=False)
        self.o_proj = HipLinear(cfg.n_heads * self.head_dim, cfg.dim, bias=False)

        self.rotary = RotaryEmbedding(dim=self.head_dim, base=cfg.rope_theta)

    def forward(
        self,
        x: torch.Tensor,
        attention_mask: Optional[torch.Tensor] = None,
        residual: Optional[torch.Tensor] = None,
    ) -> torch.Tensor:
        """GQA (model/llama.py:95-133): causal, or with `attention_mask` in its
        place (SDPA's attn_mask: bool keeps where True, a float mask is added
        to the scaled scores; broadcastable to [B, H, S, S]); attention
        dropout with p = cfg.dropout in training mode (model/llama.py:107);
        `residual` (optional) is added inside the o_proj GEMM."""
        ops.require_gpu(x)
        bsz, seq_len, _ = x.shape
        cos, sin = self.rotary.tables(seq_len, x.device, x.dtype)
        attn_dropout = float(self.dropout) if self.training else 0.0
        seed = ops.dropout_seed(x.device) if attn_dropout > 0.0 else 0
        y = LF.AttnProjFn.apply(
            x, self.q_proj.weight, self.k_proj.weight, self.v_proj.weight, cos, sin,
            self.n_heads, self.n_kv_heads, float(self.scale), attention_mask, attn_dropout, seed,
        )
        return self.o_proj(y, residual)

    @torch.no_grad()
    def forward_cached(self, x: torch.Tensor, layer: LayerCache, step: CacheStep,
                       residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        """forward() for a step's new tokens [rows, dim], whose keys and values
        go into the layer's cache and which attend over all of it (no
        gradients, no dropout; a method, so the module's own hooks do not
        run, those of o_proj do)."""
        ops.require_gpu(x)
        qkv = ops.gemm(x, LF.fused_weight([self.q_proj.weight, self.k_proj.weight, self.v_proj.weight]))
        cos, sin = self.rotary.tables(step.max_len, x.device, x.dtype, block=256)
        q = ops.kv_cache_write(qkv, layer, step, self.n_heads, cos, sin)
        return self.o_proj(ops.paged_attention(q, layer, step, self.n_heads, float(self.scale)), residual)


class SwiGLU(nn.Module):
    def __init__(self, cfg: ModelConfig) -> None:
        super().__init__()
        self.gate_proj = HipLinear(cfg.dim, cfg.ffn_dim, bias=False)
        self.up_proj = HipLinear(cfg.dim, cfg.ffn_dim, bias=False)
        self.down_proj = HipLinear(cfg.ffn_dim, cfg.dim, bias=False)
        self.dropout = nn.Dropout(cfg.dropout)

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None,
                compute_output: bool = True, dropout: bool = True) -> torch.Tensor:
        """compute_output=False (the caller only takes gradients through the
        result): the down projection's product is left uncomputed.
        dropout=False: none, in training mode too."""
        ops.require_gpu(x)
        p = float(self.dropout.p) if self.training and dropout else 0.0  # nn.Dropout on the gated activations
        seed = ops.dropout_seed(x.device) if p > 0.0 else 0
        return LF.MLPFn.apply(x, self.gate_proj.weight, self.up_proj.weight, self.down_proj.weight, residual,
                              torch.is_grad_enabled(), p, seed, compute_output)


class TransformerBlock(nn.Module):
    def __init__(self, cfg: ModelConfig) -> None:
        super().__init__()
        self.input_norm = RMSNorm(cfg.dim, eps=cfg.rms_norm_eps)
        self.attn = GroupedQueryAttention(cfg)
        self.post_attn_norm = RMSNorm(cfg.dim, eps=cfg.rms_norm_eps)
        self.mlp = SwiGLU(cfg)

    def forward(self, x: torch.Tensor, attention_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        # x + attn(norm(x)); then x + mlp(norm(x)) — residual adds in the GEMM
        # epilogues, residual gradients inside the norm backward
        h, x = self.input_norm.forward_with_residual(x)
        x = self.attn(h, attention_mask=attention_mask, residual=x)
        h, x = self.post_attn_norm.forward_with_residual(x)
        # the block's output is the MLP's: under output_unused() (the ZeRO-3
        # recompute) its value is not formed
        return self.mlp(h, residual=x, compute_output=not LF.output_is_unused())

    @torch.no_grad()
    def forward_cached(self, x: torch.Tensor, layer: LayerCache, step: CacheStep) -> torch.Tensor:
        """forward() for a step's new tokens [rows, dim] over a cache (no
        gradients, no dropout, no hooks of the block or its attention)."""
        x = self.attn.forward_cached(self.input_norm(x), layer, step, residual=x)
        return self.mlp(self.post_attn_norm(x), residual=x, dropout=False)


@dataclass
class CausalLMOutput:
    logits: Optional[torch.Tensor]
    loss: Optional[torch.Tensor] = None


class LlamaForCausalLM(nn.Module):
    def __init__(self, cfg: ModelConfig) -> None:
        super().__init__()
        self.cfg = cfg
        # construction order = the reference's (its RNG draws and parameter order)
        self.tok_embeddings = HipEmbedding(cfg.vocab_size, cfg.dim)
        self.dropout = nn.Dropout(cfg.dropout)
        self.layers = nn.ModuleList([TransformerBlock(cfg) for _ in range(cfg.n_layers)])
        self.norm = RMSNorm(cfg.dim, eps=cfg.rms_norm_eps)
        self.lm_head = HipLMHead(cfg.dim, cfg.vocab_size, bias=False)

        if cfg.tie_word_embeddings:
            self.lm_head.weight = self.tok_embeddings.weight

        self.apply(self._init_weights)
        self._zero3_executor = None
        self.loss_chunk_size = 0
        self.activation_checkpointing = False
        # training loss without returned logits: LM head and cross entropy fused
        self.fused_lm_head_loss = True

    def _init_weights(self, module: nn.Module) -> None:
        if isinstance(module, (nn.Linear, nn.Embedding)):
            nn.init.normal_(module.weight, mean=0.0, std=self.cfg.initializer_range)
            if isinstance(module, nn.Linear) and module.bias is not None:
                nn.init.zeros_(module.bias)

    def set_loss_chunk_size(self, chunk_size: int) -> None:
        if chunk_size < 0:
            raise ValueError(f"loss chunk size must be non-negative, got {chunk_size}")
        self.loss_chunk_size = int(chunk_size)

    def set_activation_checkpointing(self, enabled: bool) -> None:
        self.activation_checkpointing = bool(enabled)

    def forward(
        self,
        input_ids: torch.Tensor,
        labels: Optional[torch.Tensor] = None,
        attention_mask: Optional[torch.Tensor] = None,
        return_logits: bool = True,
    ) -> CausalLMOutput:
        if input_ids.ndim != 2:
            raise ValueError(f"input_ids should have shape [batch, seq], got {tuple(input_ids.shape)}")

        x = self._call_parametrized_module("tok_embeddings", self.tok_embeddings, input_ids)
        x = LF.dropout(x, float(self.dropout.p), self.training)

        for layer_idx in range(len(self.layers)):
            if self._should_checkpoint_activations(x):
                x = activation_checkpoint(
                    lambda hidden_states, _i=layer_idx, _m=attention_mask: self._call_layer(_i, hidden_states, _m),
                    x,
                    use_reentrant=False,
                )
            else:
                x = self._call_layer(layer_idx, x, attention_mask)

        x = self._call_parametrized_module("norm", self.norm, x)
        logits = None
        chunked = self._should_chunk_training_loss(input_ids)
        # fp16 takes the unfused loss: the fused one forms the logit gradient
        # for a unit loss gradient before the (loss-scaled) gradient arrives,
        # and (softmax - onehot) / count underflows fp16's range
        if labels is not None and not return_logits and self.fused_lm_head_loss and x.dtype != torch.float16:
            if labels.shape != input_ids.shape:
                raise ValueError(
                    f"labels should have same shape as input_ids; got {tuple(labels.shape)} vs {tuple(input_ids.shape)}"
                )
            # same divisor rule as the unfused paths: the chunked loss (and a
            # length-1 sequence) clamps the target count at 1
            clamp = chunked or input_ids.size(1) <= 1
            loss = self._call_parametrized_module("lm_head", self.lm_head, x, labels, clamp)
            return CausalLMOutput(logits=None, loss=loss)
        if labels is None or return_logits or not chunked:
            logits = self._call_parametrized_module("lm_head", self.lm_head, x)

        loss = None
        if labels is not None:
            if labels.shape != input_ids.shape:
                raise ValueError(
                    f"labels should have same shape as input_ids; got {tuple(labels.shape)} vs {tuple(input_ids.shape)}"
                )
            if logits is not None:
                loss = self._full_cross_entropy(logits=logits, labels=labels, internal=not return_logits)
            else:
                loss = self._chunked_cross_entropy(hidden_states=x, labels=labels)
            if not return_logits:
                logits = None

        return CausalLMOutput(logits=logits, loss=loss)

    def _call_layer(self, layer_idx: int, hidden_states: torch.Tensor, attention_mask: Optional[torch.Tensor]):
        layer = self.layers[layer_idx]
        return self._call_parametrized_module(f"layers.{layer_idx}", layer, hidden_states, attention_mask)

    def _should_checkpoint_activations(self, hidden_states: torch.Tensor) -> bool:
        return (
            self.activation_checkpointing
            and self.training
            and self._zero3_executor is None
            and hidden_states.requires_grad
        )

    def _should_chunk_training_loss(self, input_ids: torch.Tensor) -> bool:
        return self.loss_chunk_size > 0 and input_ids.size(1) > 1 and self._zero3_executor is None

    def _full_cross_entropy(self, logits: torch.Tensor, labels: torch.Tensor, internal: bool = False) -> torch.Tensor:
        """Mean CE of logits[:, :-1] against labels[:, 1:], ignore_index -100
        (model/llama.py:273-280).  A length-1 sequence gives a zero loss."""
        if logits.size(1) <= 1:
            return LF.cross_entropy(logits, labels, clamp=True, inplace=False)
        return LF.cross_entropy(logits, labels, clamp=False, inplace=internal)

    def _chunked_cross_entropy(self, hidden_states: torch.Tensor, labels: torch.Tensor) -> torch.Tensor:
        """Sum of per-token losses / max(#targets, 1) (model/llama.py:282-302).
        The LM head runs once over all positions; the loss kernel streams the
        logits row by row, which yields the chunked sum exactly."""
        logits = self._call_parametrized_module("lm_head", self.lm_head, hidden_states)
        return LF.cross_entropy(logits, labels, clamp=True, inplace=True)

    def _call_parametrized_module(self, module_name: str, module: nn.Module, *args: Any) -> torch.Tensor:
        executor = self._zero3_executor
        if executor is None:
            return module(*args)
        return executor.call_module(module_name, module, *args)

    def new_cache(self, batch: int, max_len: int, dtype: Optional[torch.dtype] = None, page_size: int = 64) -> KVCache:
        """A cache for `batch` sequences of up to max_len tokens, on the
        model's device; dtype torch.float8_e4m3fn stores it in 8 bits (None:
        the model's dtype)."""
        w = self.tok_embeddings.weight
        return KVCache(self.cfg.n_layers, self.cfg.n_kv_heads, self.cfg.head_dim, batch=batch,
                       n_pages=batch * -(-max_len // page_size), page_size=page_size, dtype=w.dtype, storage=dtype,
                       device=w.device)

    @torch.no_grad()
    def forward_cached(self, ids: torch.Tensor, cache: KVCache, step: Union[CacheStep, DraftStep], *,
                       rows: str = "last") -> torch.Tensor:
        """Logits [B, V] of each sequence's last new token, or of every new
        token (rows="all": [step.rows, V]); rows="none" fills the cache alone
        and returns the last block's output.  ids: the step's new tokens,
        sequence after sequence ([rows] int64); step: what cache.step(counts)
        returned for them.  Without dropout, whatever the mode; forward hooks of
        the model, its blocks and their attention do not run.  The row of a
        sequence that has no new tokens says nothing, nor do rows of no
        sequence."""
        if rows not in ("last", "all", "none"):
            raise ValueError(f"rows must be 'last', 'all' or 'none', not {rows!r}")
        if self._zero3_executor is not None and not getattr(self._zero3_executor, "params_materialized", False):
            raise RuntimeError("a ZeRO-3 sharded model has no cached forward: gather its parameters first "
                               "(summon_full_params; a forward within it hands them back) or generate without use_cache")
        if ids.dim() != 1 or ids.numel() != step.rows:
            raise ValueError(f"ids should hold the step's {step.rows} tokens, got shape {tuple(ids.shape)}")
        if step.rows == 0:
            raise ValueError("a step without new tokens has no logits")
        if len(cache.layers) != len(self.layers):
            raise ValueError(f"a cache of {len(cache.layers)} layers for a model of {len(self.layers)}")
        x = self.tok_embeddings(ids)
        for layer, block in zip(cache.layers, self.layers):
            x = block.forward_cached(x, layer, step)
        if rows == "none":
            return x
        if rows == "last":
            x = ops.embedding_fwd((step.row_start[1:] - 1).long(), x)  # rows of x
        return self.lm_head(self.norm(x))

    @torch.no_grad()
    def generate(
        self,
        input_ids: torch.Tensor,
        max_new_tokens: int,
        temperature: float = 1.0,
        top_k: Optional[int] = None,
        *,
        use_cache: bool = False,
        cache_dtype: Optional[torch.dtype] = None,
        repetition_penalty: Union[float, torch.Tensor] = 1.0,
        presence_penalty: Union[float, torch.Tensor] = 0.0,
        frequency_penalty: Union[float, torch.Tensor] = 0.0,
        logit_bias: Optional[torch.Tensor] = None,
        token_mask: Union[None, torch.Tensor, Callable[[torch.Tensor], torch.Tensor]] = None,
        draft_model: Optional["LlamaForCausalLM"] = None,
        draft_tokens: Union[int, Sequence[int]] = 4,
    ) -> torch.Tensor:
        """Autoregressive sampling with the reference's semantics
        (model/llama.py:311-335): each new token takes a full forward over the
        last max_seq_len tokens; temperature <= 0 picks the arg-max, otherwise
        the logits / temperature, cut to their top_k largest, are sampled.
        The sequence grows in one preallocated buffer.

        use_cache keeps every layer's keys and values (in cache_dtype; see
        new_cache) and runs new tokens alone through the model, as long as the
        sequence fits max_seq_len; past that the window moves, which a cache
        cannot follow, and each token takes a full forward again.  The
        penalties, logit_bias and token_mask (a mask, or a function that makes
        one of the [B, t] tokens so far) adjust the logits first, as
        ops.process_logits says, the prompt counting for repetition_penalty
        alone.  They are then looked at, for which the host waits for the
        device: a row without a token to choose (all -inf, or NaN; infinite
        where a token is sampled) is a ValueError.

        draft_model (of the same vocabulary) drafts draft_tokens tokens ahead,
        which one pass of this model then verifies: a chain that it draws from
        its own distribution, or, given widths such as (3, 2, 1), a tree of its
        likeliest tokens, that many children for each node of a level.  What is
        generated is distributed as without it (temperature <= 0: the same
        tokens, as far as the two ways to compute the logits agree).  Both
        models keep caches; the whole text has to fit both's max_seq_len, there
        are up to 4096 sequences and drafted tokens of each (the text's last one
        counts), and penalties, logit_bias and token_mask are refused."""
        if cache_dtype is not None and not use_cache and draft_model is None:
            raise ValueError("cache_dtype is for use_cache=True")
        self.eval()
        bsz, t0 = input_ids.shape
        seq = input_ids.new_empty((bsz, t0 + max_new_tokens))
        seq[:, :t0] = input_ids
        window = self.cfg.max_seq_len
        penalties = ((repetition_penalty, 1.0), (presence_penalty, 0.0), (frequency_penalty, 0.0))
        adjust = (any(torch.is_tensor(p) or p != none for p, none in penalties)
                  or logit_bias is not None or token_mask is not None)
        if draft_model is not None:
            if adjust:
                raise ValueError("penalties, logit_bias and token_mask are not taken with a draft_model")
            return self._generate_drafted(seq, t0, temperature, top_k, cache_dtype, draft_model, draft_tokens)
        prompts = torch.full((bsz,), t0, dtype=torch.int32, device=seq.device) if adjust else None
        cache, cached = None, 0
        if use_cache and 0 < t0 <= window and max_new_tokens > 0:
            cache = self.new_cache(bsz, min(t0 + max_new_tokens - 1, window), cache_dtype)
        for t in range(t0, t0 + max_new_tokens):
            if cache is not None and t <= window:
                step = cache.step([t - cached] * bsz)
                last = self.forward_cached(seq[:, cached:t].reshape(-1), cache, step)
                cached = t
            else:
                cache = None
                context = seq[:, max(0, t - window) : t].contiguous()
                last = self(context).logits[:, -1, :]
            if adjust:
                last = ops.process_logits(
                    last, tokens=seq[:, :t], prompt_lengths=prompts, repetition_penalty=repetition_penalty,
                    presence_penalty=presence_penalty, frequency_penalty=frequency_penalty, bias=logit_bias,
                    mask=token_mask(seq[:, :t]) if callable(token_mask) else token_mask)
                _require_choice(last, t, temperature)
            seq[:, t] = _next_token(last.float(), temperature, top_k)
        return seq

    def _generate_drafted(self, seq: torch.Tensor, t0: int, temperature: float, top_k: Optional[int],
                          cache_dtype: Optional[torch.dtype], draft: "LlamaForCausalLM",
                          draft_tokens: Union[int, Sequence[int]]) -> torch.Tensor:
        """generate() with a draft model; seq: [B, t0 + new], its first t0 given."""
        chain = isinstance(draft_tokens, numbers.Integral)  # NumPy's too
        widths = [1] * int(draft_tokens) if chain else [int(w) for w in draft_tokens]
        B, total = seq.shape
        if not widths or min(widths) < 1:
            raise ValueError(f"draft_tokens must be positive, got {draft_tokens}")
        if draft.cfg.vocab_size != self.cfg.vocab_size:
            raise ValueError(f"a draft model of {draft.cfg.vocab_size} tokens for one of {self.cfg.vocab_size}")
        if t0 < 1 or total > min(self.cfg.max_seq_len, draft.cfg.max_seq_len):
            raise ValueError(f"{total} tokens (of which {t0} are given) do not fit both models' max_seq_len "
                             f"({self.cfg.max_seq_len} and {draft.cfg.max_seq_len})")
        if not chain and max(widths) > self.cfg.vocab_size:
            raise ValueError(f"{max(widths)} children of a node from {self.cfg.vocab_size} tokens")
        nodes = 1 + sum(itertools.accumulate(widths, operator.mul))
        if B > DraftCache.MOST or nodes > DraftCache.MOST:
            raise ValueError(f"{B} sequences with a draft of {nodes} tokens each (the root among them): up to "
                             f"{DraftCache.MOST} of both are taken with a draft_model")
        if total == t0:
            return seq
        draft.eval()
        tree, dev = _Tree(widths), seq.device
        N, models = tree.nodes, (self, draft)
        page = 64
        caches = [DraftCache(m.cfg.n_layers, m.cfg.n_kv_heads, m.cfg.head_dim, batch=B,
                             n_pages=B * -(-(total + N) // page), page_size=page, dtype=m.tok_embeddings.weight.dtype,
                             storage=cache_dtype, device=dev, max_len=total + N) for m in models]
        if t0 > 1:
            for m, cache in zip(models, caches):
                step = cache.step([t0 - 1] * B, max_len=t0 - 1)
                m.forward_cached(seq[:, : t0 - 1].reshape(-1), cache, step, rows="none")
        parents = None if chain else torch.tensor(tree.parents, dtype=torch.int32, device=dev)
        new = torch.full((B,), N, dtype=torch.int32, device=dev)
        cached = torch.full((B,), t0 - 1, dtype=torch.int32, device=dev)  # tokens before the root
        lengths = [t0] * B  # of the texts
        drawn = chain and temperature > 0
        i = torch.arange(N, device=dev)
        text = torch.nn.functional.pad(seq, (0, N))  # room for what is cut off at the end
        while min(lengths) < total:
            bound = dict(rows=B * N, max_new=N, max_len=max(lengths) - 1 + N, keep=cached, parents=parents)
            ids = torch.empty((B, N), dtype=torch.int64, device=dev)
            ids[:, 0] = text.gather(1, cached.long()[:, None])[:, 0]
            probs: List[torch.Tensor] = []
            ahead = caches[1].step(new, **bound)
            for level, (lo, hi) in enumerate(tree.levels):
                step, last = tree.step_of(ahead, level), level == len(tree.widths)
                x = draft.forward_cached(ids[:, lo:hi].reshape(-1), caches[1], step, rows="none" if last else "all")
                if last:
                    break
                if drawn:  # logits that have no softmax draw from all alike (drawing from NaN would end the process)
                    law = torch.softmax(_cut(x.float() / temperature, top_k), -1)
                    probs.append(law.nan_to_num_(nan=1.0 / law.size(-1)))
                    ids[:, hi] = torch.multinomial(probs[-1], 1)[:, 0]
                else:
                    first, end = tree.levels[level + 1]
                    ids[:, first:end] = x.topk(tree.widths[level]).indices.view(B, -1)
            step = caches[0].step(new, **bound)
            flat = ids.view(-1)
            logits = self.forward_cached(flat, caches[0], step, rows="all")
            if temperature > 0:
                logits = _cut(logits.float(), top_k) if top_k is not None else logits
            q = torch.stack([probs[0], *probs], 1).view(B * N, -1) if drawn else None  # the root's is not read
            counts, kept, chosen = ops.verify_draft(
                logits, flat, step.row_start, N, torch.rand(B * N, dtype=torch.float64, device=dev),
                temperature=float(max(temperature, 0.0)), parents=parents, draft_probs=q)
            # no further than the text goes; the last token of what is gained is the next root
            counts = torch.minimum(counts, (total - 1 - cached).clamp(min=0))
            if not chain:
                for cache, made in zip(caches, (step, ahead)):
                    cache.keep(made, kept, counts)
            at = cached.long()[:, None] + 1 + i
            gained = i < counts[:, None]
            text.scatter_(1, at, torch.where(gained, chosen, text.gather(1, at)))
            cached = cached + counts
            *ends, none = torch.cat([cached, (gained & (chosen < 0)).any().view(1)]).tolist()  # waits, once a step
            if none:
                raise ValueError("a row's logits leave no token to choose (NaN, or infinite where it is sampled)")
            lengths = [n + 1 for n in ends]
        return text[:, :total].contiguous()
