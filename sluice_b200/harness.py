"""A DeepSeek-V2-Lite-shaped decoder around the offloaded MoE layers.

The reference's headline numbers are whole-model decode tok/s inside vLLM;
this harness gives the MoE hot path the same surroundings at the shapes the
workload names (random-init bf16, no checkpoint): token embedding, 27
decoder layers of [RMSNorm -> multi-head latent attention -> residual ->
RMSNorm -> FFN -> residual] with a dense SwiGLU FFN in layer 0 and an MoE
layer elsewhere, final RMSNorm, the vocabulary head and greedy sampling.

The MoE layers are this package's hot path (``SluiceMoELayer``: router,
device slot planner, expert streamer, tcgen05 fused experts). Around them,
on a CUDA device, the attention core, each residual add + RMSNorm and (for
one or two sequences) the projections are also this package's kernels
(``sl_mla_decode``, ``sl_add_rmsnorm``, ``sl_linear_small``); the rest is
PyTorch (cuBLAS GEMMs): it is the harness around the hot path, not part of
it. The same module runs on the host for the CPU baseline, with PyTorch ops
throughout and the MoE layers replaced by the oracle's torch-native MoE and
slot policy.

Attention is decode-only MLA in its absorbed form over a compressed cache
(kv_lora_rank 512 latent + 64 rotary dims per token and layer): per token
``q`` (16 heads x (128 nope + 64 rope)), the latent ``c_kv`` (RMSNormed) and
``k_pe`` (rotary) are written at the sequence's position; scores are
``q_nope W_uk . c_kv + q_pe . k_pe`` over every cached position (fixed
shapes, masked beyond the sequence's length, so a step captures in one CUDA
graph); the output is ``softmax . c_kv`` projected through ``W_uv`` and the
output projection. Prompts go through the same decode step, one position per
step, or (``prefill``, on a CUDA device) whole or in chunks through the prompt
pass (``sluice_b200.prompt``): the block planner's slot maps, rotary positions
in place, keys and values expanded from the latents, causal attention over the
packed sequences. The cache is one run of ``max_len`` rows per sequence, or a
pool of blocks that the sequences share (``cache_blocks``). Rotary embedding: RoPE (theta 10000) on adjacent dim
pairs. In the PyTorch form the causal mask is an additive bias folded into
the score GEMM; the fused kernel reads each sequence's positions 0..P.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch
import torch.nn.functional as F

from .configs import V2_LITE, MoEConfig


@dataclass(frozen=True)
class DecoderConfig:
    moe: MoEConfig
    num_layers: int
    first_dense: int          # leading layers with a dense FFN
    dense_intermediate: int
    num_heads: int
    kv_lora_rank: int
    qk_nope: int
    qk_rope: int
    v_head: int
    vocab: int
    rms_eps: float = 1e-6
    rope_theta: float = 10000.0

    @property
    def hidden(self) -> int:
        return self.moe.hidden

    @property
    def num_moe_layers(self) -> int:
        return self.num_layers - self.first_dense


V2_LITE_DECODER = DecoderConfig(
    moe=V2_LITE, num_layers=27, first_dense=1, dense_intermediate=10944, num_heads=16,
    kv_lora_rank=512, qk_nope=128, qk_rope=64, v_head=128, vocab=102400)


def _rms(x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    return F.rms_norm(x, (x.shape[-1],), w, eps)


def _rope(x: torch.Tensor, freqs: torch.Tensor) -> torch.Tensor:
    """RoPE on the last dim of x [B, ..., R] (pairs of adjacent dims rotated
    as complex numbers) by freqs [B, R/2] (complex64)."""
    shape = [freqs.shape[0]] + [1] * (x.dim() - 2) + [freqs.shape[1]]
    xc = torch.view_as_complex(x.float().reshape(*x.shape[:-1], -1, 2))
    return torch.view_as_real(xc * freqs.view(shape)).flatten(-2).to(x.dtype)


class DecoderHarness:
    """Greedy decode of ``batch`` sequences through the decoder; ``moe(li,
    x)`` computes MoE layer ``li`` (0-based over the MoE layers) of normed
    hidden states ``x`` [batch, H]."""

    def __init__(self, cfg: DecoderConfig, moe, batch: int, max_len: int, seed: int = 0,
                 device="cuda", std: float = 0.02, fused_attention: bool | None = None,
                 cache_blocks: int | None = None, block_size: int = 64):
        """``fused_attention`` (default: on a CUDA device) runs each layer's
        attention core as the library's one-launch MLA decode kernel
        (``sl_mla_decode``) and each residual add with the RMSNorm after it
        as one launch (``sl_add_rmsnorm``); otherwise, and on the host, as
        PyTorch ops.

        ``cache_blocks`` gives the sequences a shared pool of so many blocks
        of ``block_size`` positions (a multiple of 32) per layer instead of
        ``max_len`` rows each; they take blocks as they grow, up to
        ``max_len`` positions, and ``reset`` returns them
        (``check_blocks`` raises if the pool ran out)."""
        self.cfg = cfg
        self.moe = moe
        self.batch = batch
        self.max_len = max_len
        self.device = torch.device(device)
        dev, bf = self.device, torch.bfloat16
        # seeded on the device that holds the weights (the host port draws
        # its own values: it is timed, not compared)
        g = torch.Generator(device=dev)
        g.manual_seed(seed * 7919 + 17)
        H, nh = cfg.hidden, cfg.num_heads
        dq = cfg.qk_nope + cfg.qk_rope

        def w(*shape):
            return (torch.randn(*shape, generator=g, device=dev) * std).to(bf)

        self.embed = w(cfg.vocab, H)
        self.head = w(cfg.vocab, H)
        self.final_norm = torch.ones(H, dtype=bf, device=dev)
        self.layers = []
        for li in range(cfg.num_layers):
            lw = {
                "in_norm": torch.ones(H, dtype=bf, device=dev),
                "post_norm": torch.ones(H, dtype=bf, device=dev),
                "kv_norm": torch.ones(cfg.kv_lora_rank, dtype=bf, device=dev),
                # q_proj [nh * dq, H] and kv_a_proj [rank + rope, H] as one GEMM
                "wqkv": w(nh * dq + cfg.kv_lora_rank + cfg.qk_rope, H),
                # kv_b_proj [nh * (nope + v), rank] split per head into the
                # absorbed key (W_uk) and value (W_uv) maps
                "w_uk": w(nh, cfg.qk_nope, cfg.kv_lora_rank),
                "w_uv": w(nh, cfg.v_head, cfg.kv_lora_rank),
                "wo": w(H, nh * cfg.v_head),
            }
            if li < cfg.first_dense:
                lw["w13"] = w(2 * cfg.dense_intermediate, H)
                lw["w2"] = w(H, cfg.dense_intermediate)
            self.layers.append(lw)
        L = cfg.num_layers
        # compressed cache per layer and position: [c_kv (rank) | k_pe (rope)]
        self.paged = cache_blocks is not None
        if self.paged:
            if block_size <= 0 or block_size % 32 or cache_blocks <= 0:
                raise ValueError("a paged cache needs blocks of a multiple of 32 positions")
            rows = (cache_blocks, block_size)
            self.block_size = block_size
            self.block_table = torch.full((batch, -(-max_len // block_size)), -1,
                                          dtype=torch.int32, device=dev)
            self.free_blocks = torch.arange(cache_blocks, dtype=torch.int32, device=dev)
            self.free_range = torch.tensor([0, cache_blocks], device=dev)
        else:
            # every sequence owns one block of max_len rows
            rows = (batch, max_len)
            self.block_size = max_len
            self.block_table = torch.arange(batch, dtype=torch.int32, device=dev)[:, None]
            self.free_blocks = self.free_range = None
        self.cache = torch.zeros(L, *rows, cfg.kv_lora_rank + cfg.qk_rope, dtype=bf, device=dev)
        self.kv_status = torch.zeros((), dtype=torch.int32, device=dev)
        self._ones = torch.ones(batch, dtype=torch.int32, device=dev)
        # angles in 64 bits, as the prompt pass forms them: both write one cache
        inv = cfg.rope_theta ** (torch.arange(0, cfg.qk_rope, 2).double() / -cfg.qk_rope)
        ang = torch.arange(max_len).double()[:, None] * inv[None, :]
        self.freqs = torch.polar(torch.ones_like(ang), ang).to(torch.complex64).to(dev)
        self.rope_cs = torch.view_as_real(self.freqs).contiguous()    # [max_len, r/2, 2]
        self.fused_attention = (self.device.type == "cuda") if fused_attention is None \
            else bool(fused_attention)
        if self.paged and not self.fused_attention:
            raise ValueError("a paged cache needs the fused attention")
        self._rotary = None   # of the prompt pass, made with its first prompt
        self.pos = torch.zeros(batch, dtype=torch.long, device=dev)
        self.scale = 1.0 / math.sqrt(dq)
        self._ar = torch.arange(max_len, device=dev)
        self._rows = torch.arange(batch, device=dev)
        # w_uk / w_uv per head, laid out for batched GEMMs over heads
        for lw in self.layers:
            lw["w_uk_t"] = lw["w_uk"].contiguous()                  # [nh, nope, rank]
            lw["w_uv_t"] = lw["w_uv"].transpose(1, 2).contiguous()  # [nh, rank, v]

    def reset(self) -> None:
        self.pos.zero_()
        if self.paged:
            self.block_table.fill_(-1)
            torch.arange(self.free_blocks.numel(), out=self.free_blocks)
            self.free_range[0] = 0
            self.free_range[1] = self.free_blocks.numel()
        self.kv_status.zero_()

    def _plan(self, context: torch.Tensor, new: torch.Tensor, tokens: int, kv_tokens: int = 0):
        from .prompt import plan_kv_blocks
        plan = plan_kv_blocks(context, new, self.block_table, self.free_blocks, self.free_range,
                              self.block_size, tokens, num_kv_tokens=kv_tokens)
        torch.maximum(self.kv_status, plan.status[0], out=self.kv_status)
        return plan

    _BLOCKS = ("block_table", "free_blocks", "free_range", "kv_status")

    def save_blocks(self) -> dict:
        """Copies of what the block planner keeps."""
        return {n: getattr(self, n).clone() for n in self._BLOCKS if getattr(self, n) is not None}

    def restore_blocks(self, saved: dict) -> None:
        for n, t in saved.items():
            getattr(self, n).copy_(t)

    def check_blocks(self) -> None:
        """Raise if a step since ``reset`` found no block for a position, or
        no room below ``max_len``, on either cache (synchronises)."""
        from .prompt import KvPlanError
        status = int(self.kv_status.item())
        if status:
            raise KvPlanError(status)

    def _attention(self, li: int, x: torch.Tensor, mask_bias: torch.Tensor | None,
                   freqs: torch.Tensor | None) -> torch.Tensor:
        cfg, lw = self.cfg, self.layers[li]
        B, nh, R = x.shape[0], cfg.num_heads, cfg.kv_lora_rank
        dq = cfg.qk_nope + cfg.qk_rope
        qkv = self._linear(x, lw["wqkv"])
        if self.fused_attention:
            from ._lib import check, lib, ptr
            o = torch.empty(B, nh * cfg.v_head, dtype=x.dtype, device=x.device)
            if self.paged:
                cache, table = self.cache[li], self.block_table
                check(lib().sl_mla_decode_paged(
                    ptr(qkv), qkv.shape[1], ptr(lw["kv_norm"]), cfg.rms_eps, ptr(lw["w_uk_t"]),
                    ptr(lw["w_uv"]), ptr(self.rope_cs), ptr(self.pos), ptr(cache),
                    cache.shape[0], self.block_size, ptr(table), table.shape[1], table.shape[1],
                    B, nh, cfg.qk_nope, cfg.qk_rope, R, cfg.v_head, self.max_len, self.scale,
                    ptr(o), torch.cuda.current_stream().cuda_stream), "sl_mla_decode_paged")
                return self._linear(o, lw["wo"])
            check(lib().sl_mla_decode(ptr(qkv), qkv.shape[1], ptr(lw["kv_norm"]), cfg.rms_eps,
                                      ptr(lw["w_uk_t"]), ptr(lw["w_uv"]), ptr(self.rope_cs),
                                      ptr(self.pos), ptr(self.cache[li]), B, nh, cfg.qk_nope,
                                      cfg.qk_rope, R, cfg.v_head, self.max_len, self.scale,
                                      ptr(o), torch.cuda.current_stream().cuda_stream),
                  "sl_mla_decode")
            return self._linear(o, lw["wo"])
        q = qkv[:, :nh * dq].view(B, nh, dq)
        kv = qkv[:, nh * dq:]
        c = _rms(kv[:, :R], lw["kv_norm"], cfg.rms_eps)
        k_pe = _rope(kv[:, R:], freqs)
        self.cache[li, self._rows, self.pos] = torch.cat([c, k_pe], dim=-1)
        # absorbed query: [q_nope W_uk | rope(q_pe)] against [c_kv | k_pe]
        q_lat = torch.bmm(q[..., :cfg.qk_nope].transpose(0, 1), lw["w_uk_t"])  # [nh, B, R]
        qf = torch.cat([q_lat.transpose(0, 1), _rope(q[..., cfg.qk_nope:], freqs)], dim=-1)
        cl = self.cache[li]                                                   # [B, Lmax, R+r]
        s = torch.baddbmm(mask_bias, qf, cl.transpose(1, 2), alpha=self.scale)
        p = torch.softmax(s, dim=-1)
        o_lat = torch.bmm(p, cl[..., :R])                                     # [B, nh, R]
        o = torch.bmm(o_lat.transpose(0, 1), lw["w_uv_t"])                   # [nh, B, v]
        return F.linear(o.transpose(0, 1).reshape(B, nh * cfg.v_head), lw["wo"])

    def _linear(self, x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
        """x @ w.T: the library's skinny linear (``sl_linear_small``) for
        one or two rows on the device (faster than cuBLAS there), else
        PyTorch's (cuBLAS)."""
        if self.fused_attention and x.shape[0] <= 2 and x.shape[1] * x.shape[0] * 2 <= 200 * 1024:
            from ._lib import check, lib, ptr
            x = x.contiguous()
            y = torch.empty(x.shape[0], w.shape[0], dtype=x.dtype, device=x.device)
            check(lib().sl_linear_small(ptr(x), x.shape[0], x.shape[1], ptr(w), w.shape[0],
                                        ptr(y), torch.cuda.current_stream().cuda_stream),
                  "sl_linear_small")
            return y
        return F.linear(x, w)

    def _add_norm(self, h: torch.Tensor, delta: torch.Tensor | None,
                  w: torch.Tensor) -> torch.Tensor:
        """h += delta (in place; None: no add), then RMSNorm(h) * w."""
        eps = self.cfg.rms_eps
        if self.fused_attention:
            from ._lib import check, lib, ptr
            out = torch.empty_like(h)
            check(lib().sl_add_rmsnorm(ptr(h), ptr(delta) if delta is not None else None,
                                       ptr(w), eps, ptr(out), h.shape[0], h.shape[1],
                                       torch.cuda.current_stream().cuda_stream),
                  "sl_add_rmsnorm")
            return out
        if delta is not None:
            h.add_(delta)
        return _rms(h, w, eps)

    def _dense_ffn(self, li: int, x: torch.Tensor) -> torch.Tensor:
        lw = self.layers[li]
        g, u = F.linear(x, lw["w13"]).chunk(2, dim=-1)
        return F.linear(F.silu(g) * u, lw["w2"])

    def step(self, ids: torch.Tensor) -> torch.Tensor:
        """One decode step: token ids [batch] at the sequences' positions ->
        the greedy next ids [batch]; the positions advance by one."""
        cfg = self.cfg
        h = self.embed[ids]
        if self.paged:
            self._plan(self.pos.to(torch.int32), self._ones, self.batch)
        freqs = mask_bias = None
        if self.fused_attention:
            # (KV_PLAN_NO_BLOCKS is 1; the kernel stays within max_len)
            torch.maximum(self.kv_status, (self.pos >= self.max_len).any(), out=self.kv_status)
        else:
            # per step: the positions' rotations and the causal mask as an additive
            # bias over the cache (0 up to each sequence's position, -inf after)
            freqs = self.freqs[self.pos]
            mask_bias = torch.zeros(h.shape[0], 1, self.max_len, dtype=h.dtype, device=h.device)
            mask_bias.masked_fill_((self._ar[None, :] > self.pos[:, None])[:, None, :],
                                   float("-inf"))
        x = self._add_norm(h, None, self.layers[0]["in_norm"])
        for li in range(cfg.num_layers):
            lw = self.layers[li]
            x = self._add_norm(h, self._attention(li, x, mask_bias, freqs), lw["post_norm"])
            f = self._dense_ffn(li, x) if li < cfg.first_dense else \
                self.moe(li - cfg.first_dense, x)
            nxt = self.layers[li + 1]["in_norm"] if li + 1 < cfg.num_layers else self.final_norm
            x = self._add_norm(h, f, nxt)
        logits = F.linear(x, self.head)
        self.pos.add_(1)
        return logits.argmax(dim=-1)

    def _prompt_attention(self, li: int, x: torch.Tensor, plan, has_context: bool,
                          status: torch.Tensor) -> torch.Tensor:
        """The attention of packed prompt rows x [T, H]: their latents and
        rotated keys go to the cache, keys and values are expanded from the
        latents of the whole sequences (the cached beginnings included).
        ``status`` is raised where a wait of the kernel ran out."""
        from .prompt import prompt_attention
        cfg, lw = self.cfg, self.layers[li]
        nh, R = cfg.num_heads, cfg.kv_lora_rank
        dq = cfg.qk_nope + cfg.qk_rope
        T = x.shape[0]
        qkv = F.linear(x, lw["wqkv"])
        q, k_pe = qkv[:, :nh * dq].view(T, nh, dq), qkv[:, nh * dq + R:].view(T, 1, cfg.qk_rope)
        self._rotary(plan.positions, q, k_pe, q_offset=cfg.qk_nope, out_q=q, out_k=k_pe)
        c = _rms(qkv[:, nh * dq:nh * dq + R], lw["kv_norm"], cfg.rms_eps)
        rows = torch.cat([c, k_pe[:, 0]], dim=-1)
        cache = self.cache[li].flatten(0, 1)
        cache.index_copy_(0, plan.slots, rows)
        if has_context:
            rows = cache[plan.kv_slots]
        if "w_ukv" not in lw:
            # W_uk and W_uv of each head as one map from the latent
            lw["w_ukv"] = torch.cat([lw["w_uk"], lw["w_uv"]], dim=1).flatten(0, 1)
        kv = F.linear(rows[:, :R], lw["w_ukv"]).view(-1, nh, cfg.qk_nope + cfg.v_head)
        o = prompt_attention(q, kv[..., :cfg.qk_nope], kv[..., cfg.qk_nope:], plan.cu_new,
                             plan.cu_total, k_shared=rows[:, R:], scale=self.scale,
                             status=status)
        return F.linear(o.flatten(1), lw["wo"])

    def prefill(self, ids: torch.Tensor, lengths: list[int],
                context: list[int] | None = None) -> torch.Tensor:
        """Prompts, or the next chunks of prompts, in one pass: ``ids`` [T] are
        the sequences' tokens one after the other, ``lengths`` [batch] how many
        each has (0: none in this pass). They continue at the sequences'
        positions, which advance by ``lengths``. Returns the greedy next ids
        [batch] behind each sequence's last token (-1 for a sequence without
        tokens). ``context`` are the positions, where the caller knows them;
        otherwise they are read back. Raises ``KvPlanError``, with nothing
        changed, where the pool has too few blocks left or a position before
        the new tokens has none, and ``SluiceError`` where a layer's attention
        gave up on a wait; an error, of the MoE layers too, moves no position
        and takes no block. CUDA with the fused attention only; the MoE layers
        take the pass as one step of T rows."""
        if not self.fused_attention:
            raise ValueError("prefill runs on a CUDA device with the fused attention")
        from ._lib import KV_PLAN_BAD_INPUT
        from .prompt import KvPlanError
        cfg, dev = self.cfg, self.device
        if len(lengths) != self.batch or any(n < 0 for n in lengths):
            raise ValueError(f"lengths must be {self.batch} counts")
        T = sum(lengths)
        if tuple(ids.shape) != (T,):
            raise ValueError(f"ids must hold the {T} tokens of lengths, got {tuple(ids.shape)}")
        if context is None:
            context = self.pos.tolist()
        elif len(context) != self.batch:
            raise ValueError(f"context must be {self.batch} positions")
        if any(c + n > self.max_len for c, n in zip(context, lengths)):
            raise ValueError(f"a sequence would pass max_len {self.max_len}")
        if T == 0:
            return torch.full((self.batch,), -1, dtype=torch.long, device=dev)
        if self._rotary is None:
            from .prompt import Rotary
            self._rotary = Rotary(cfg.qk_rope, base=cfg.rope_theta, interleaved=True, device=dev)
        new = torch.tensor(lengths, dtype=torch.int32, device=dev)
        # sequences without tokens in this pass have no keys in it either
        seen = [c if n else 0 for c, n in zip(context, lengths)]
        has_context = any(seen)
        # (kept apart until the plan is known to hold: a position without a
        # block has no cache row to write)
        blocks0 = self.save_blocks()
        plan = self._plan(torch.tensor(seen, dtype=torch.int32, device=dev), new, T,
                          T + sum(seen) if has_context else 0)
        try:
            plan.check()
            # positions that the caller's context or an earlier step without a
            # block left without a cache row
            rows = plan.slots if plan.kv_slots is None else torch.cat([plan.slots, plan.kv_slots])
            if int(rows.min()) < 0:
                raise KvPlanError(KV_PLAN_BAD_INPUT)
            nxt = self._prompt_pass(ids, lengths, plan, has_context)
        except BaseException:
            self.restore_blocks(blocks0)
            raise
        self.pos.add_(new)
        return nxt

    def _prompt_pass(self, ids: torch.Tensor, lengths: list[int], plan,
                     has_context: bool) -> torch.Tensor:
        """The layers over the packed rows of a plan that holds."""
        from ._lib import check
        cfg = self.cfg
        status = torch.zeros(1, dtype=torch.int32, device=self.device)
        h = self.embed[ids]
        x = self._add_norm(h, None, self.layers[0]["in_norm"])
        for li in range(cfg.num_layers):
            lw = self.layers[li]
            x = self._add_norm(h, self._prompt_attention(li, x, plan, has_context, status),
                               lw["post_norm"])
            f = self._dense_ffn(li, x) if li < cfg.first_dense else \
                self.moe(li - cfg.first_dense, x)
            last = self.layers[li + 1]["in_norm"] if li + 1 < cfg.num_layers else self.final_norm
            x = self._add_norm(h, f, last)
        live = [b for b, n in enumerate(lengths) if n]
        ends = plan.cu_new[1:].long()[live] - 1
        nxt = torch.full((self.batch,), -1, dtype=torch.long, device=self.device)
        nxt[live] = F.linear(x[ends], self.head).argmax(dim=-1)
        check(int(status), "prompt_attention")
        return nxt


class OffloadedDecoder:
    """The decoder on this GPU with its MoE layers behind slot caches: the
    layers of a ``MoEDecodeStack`` (one GPU) or an ``EPDecodeStack``
    (expert parallelism: every rank decodes its own sequences, the MoE
    layers exchange tokens with the other ranks). A decode step replays as
    one CUDA graph that also feeds its greedy ids back as the next input."""

    def __init__(self, cfg: DecoderConfig, stack, batch: int, max_len: int, seed: int = 0,
                 cache_blocks: int | None = None, block_size: int = 64):
        self.cfg = cfg
        self.stack = stack
        self.device = stack.device
        layers = stack.layers
        if len(layers) != cfg.num_moe_layers:
            raise ValueError(f"{len(layers)} MoE layers for a decoder with {cfg.num_moe_layers}")
        self.layers = layers          # the MoE layers (slot caches, stream timers)
        self.model = DecoderHarness(cfg, lambda li, x: layers[li](x), batch, max_len, seed,
                                    self.device, cache_blocks=cache_blocks,
                                    block_size=block_size)
        self.graph = None
        self._ids = torch.zeros(batch, dtype=torch.long, device=self.device)
        self._out = None

    def _step(self) -> torch.Tensor:
        out = self.model.step(self._ids)
        self._ids.copy_(out)
        return out

    def capture(self, tokens: int | None = None) -> bool:
        """Capture one decode step (after one eager warm-up step, whose
        position is then rewound)."""
        ids0 = self._ids.clone()
        blocks0 = self.model.save_blocks()
        s = torch.cuda.Stream(self.device)
        s.wait_stream(torch.cuda.current_stream(self.device))
        with torch.cuda.stream(s):
            self._step()
        torch.cuda.current_stream(self.device).wait_stream(s)
        self.model.pos.sub_(1)
        self.model.restore_blocks(blocks0)
        self._ids.copy_(ids0)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            self._out = self._step()
        self.graph = g
        return True

    def replay(self, ids: torch.Tensor | None = None) -> torch.Tensor:
        """One decode step; ``ids`` [batch] (device) are the input tokens, or
        None to continue from the last step's greedy ids. Returns the next
        ids [batch] (a static buffer)."""
        if ids is not None:
            self._ids.copy_(ids, non_blocking=True)
        self.graph.replay()
        return self._out

    def decode_step(self, ids_host: torch.Tensor, out_host: torch.Tensor) -> torch.Tensor:
        """Public end-to-end call: host token ids in, host next ids out."""
        out_host.copy_(self.replay(ids_host.to(self.device, non_blocking=True)),
                       non_blocking=True)
        return out_host

    def prefill(self, ids: torch.Tensor, lengths: list[int],
                context: list[int] | None = None) -> torch.Tensor:
        """Prompts, or their next chunks, in one pass
        (``DecoderHarness.prefill``; the MoE layers' steps beyond the slot
        envelope run in expert waves); the sequences that had tokens go on
        from their greedy next ids. One GPU only."""
        from .ep import EPDecodeStack
        if isinstance(self.stack, EPDecodeStack):
            # (its exchanges want the same number of rows on every rank)
            raise ValueError("prefill takes the MoE layers of one GPU, not an EPDecodeStack")
        nxt = self.model.prefill(ids, lengths, context)
        self._ids.copy_(torch.where(nxt >= 0, nxt, self._ids))
        return nxt

    def save(self) -> dict:
        """The sequences' state (KV caches and their blocks, positions, next
        input ids)."""
        m = self.model
        return {"cache": m.cache.clone(), "pos": m.pos.clone(), "ids": self._ids.clone(),
                "blocks": m.save_blocks()}

    def restore(self, saved: dict) -> None:
        m = self.model
        if m.paged and "blocks" not in saved:
            raise ValueError("the state of a paged cache holds its blocks")
        m.cache.copy_(saved["cache"])
        m.pos.copy_(saved["pos"])
        self._ids.copy_(saved["ids"])
        m.restore_blocks(saved.get("blocks", {}))

    def check(self) -> None:
        self.stack.check()
        self.model.check_blocks()

    def stats(self) -> dict:
        return self.stack.stats()

    def release(self) -> None:
        self.graph = None
        if hasattr(self.stack, "release"):
            self.stack.release()
