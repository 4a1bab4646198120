"""Decode steps of an FP8 decoder on one B200: the block-scaled and paged operators as a server runs them.

The reference times a decoder's dense projections alone
(profiling/dense_qwen/bench_dense_proj.py:55-65, 80-150). This harness runs the whole
layer for one new token per sequence, at those sizes (hidden 5120, 40 query and 8 KV
heads of 128, FFN 17408):

  add_rmsnorm_quant(fp8_block) -> fp8_block_gemm (QKV, bias) -> rotary embedding
  -> paged_kv_append -> paged_decode_attention -> fp8_block_gemm_dynamic (O)
  -> add_rmsnorm_quant(fp8_block) -> fp8_block_gemm (gate, up) -> silu(gate) * up
  -> fp8_block_gemm_dynamic (down)

The rotary embedding and the gate are torch's. Lengths, page table and slots live on
the device and a step reads nothing back, so ``Decoder.step`` is captured once in a CUDA
graph and replayed for every token. Weights are random N(0, 0.02), e4m3 with one scale
per 128 x 128 block, distinct per layer.

    python cache-barrier_b200/harness/decode_layer.py --batches 1,16,64 --context 4096 --out decode_layer.json
"""

from __future__ import annotations

import argparse
import os
import sys
from dataclasses import dataclass

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, HERE)

from common import ClockSampler, gpu_info, graph_time_us, save_json  # noqa: E402

import torch  # noqa: E402

FP8 = torch.float8_e4m3fn


@dataclass(frozen=True)
class Dims:
    hidden: int = 5120
    heads: int = 40
    kv_heads: int = 8
    head_dim: int = 128
    inter: int = 17408
    eps: float = 1e-6
    rope_base: float = 1e6

    @property
    def qkv(self) -> int:
        return (self.heads + 2 * self.kv_heads) * self.head_dim


def block_weight(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """[N, K] as e4m3 and fp32 scales per 128 x 128 block, on w's device
    (``wformat.quantize_fp8_block`` does the same on the host)."""
    N, K = w.shape
    nb, kb = -(-N // 128), -(-K // 128)
    full = torch.zeros(nb * 128, kb * 128, device=w.device, dtype=torch.float32)
    full[:N, :K] = w
    t = full.view(nb, 128, kb, 128)
    s = (t.abs().amax(dim=(1, 3)) / 448.0).clamp_min(1.0 / (448.0 * 512.0))
    q = (t / s[:, None, :, None]).reshape(full.shape)[:N, :K].contiguous().to(FP8)
    return q, s


class Layer:
    """One layer's operands: (e4m3 weight, block scales) per projection."""

    def __init__(self, d: Dims, seed: int, device, dtype=torch.bfloat16):
        g = torch.Generator(device=device).manual_seed(seed)

        def rand(*shape):
            return torch.randn(*shape, generator=g, device=device)

        shapes = {"qkv": (d.qkv, d.hidden), "o": (d.hidden, d.heads * d.head_dim), "gate_up": (2 * d.inter, d.hidden),
                  "down": (d.hidden, d.inter)}
        for name, (n, k) in shapes.items():
            setattr(self, name, block_weight(0.02 * rand(n, k)))
        self.qkv_bias = (0.02 * rand(d.qkv)).to(dtype)
        self.norm_in, self.norm_mid = ((1.0 + 0.1 * rand(d.hidden)).to(dtype) for _ in range(2))

    def weight_bytes(self) -> int:
        return sum(q.numel() + 4 * s.numel() for q, s in (self.qkv, self.o, self.gate_up, self.down))


class PagedCache:
    """Keys and values of one layer, [pages, page_size, kv_heads, head_dim]."""

    def __init__(self, d: Dims, pages: int, page_size: int, device, dtype):
        shape = (pages, page_size, d.kv_heads, d.head_dim)
        self.k, self.v = (torch.zeros(shape, device=device, dtype=torch.uint8 if dtype == FP8 else dtype) for _ in range(2))
        if dtype == FP8:
            self.k, self.v = self.k.view(FP8), self.v.view(FP8)
            self.k_scale, self.v_scale = (torch.full((d.kv_heads,), 2.0 ** -4, device=device) for _ in range(2))
        else:
            self.k_scale = self.v_scale = None


@dataclass(frozen=True)
class Place:
    """Where a step's tokens stand, one entry per sequence."""

    slots: torch.Tensor  # cache slot, -1: none
    held: torch.Tensor  # tokens to attend to, the new one included
    cos: torch.Tensor  # rotary factors of the position
    sin: torch.Tensor


def rope(x: torch.Tensor, at: Place) -> torch.Tensor:
    """x [B, heads, D], rotated by each sequence's position."""
    a, b = x.float().chunk(2, dim=-1)
    return torch.cat([a * at.cos - b * at.sin, b * at.cos + a * at.sin], dim=-1).to(x.dtype)


class Decoder:
    """``layers`` layers over a batch whose sequences hold ``lens`` tokens each."""

    def __init__(self, d: Dims, layers: int, lens: list[int], max_len: int, page_size: int = 64, device="cuda",
                 dtype=torch.bfloat16, cache_dtype=None, seed: int = 0):
        if max(lens) >= max_len:
            raise ValueError(f"a sequence of {max(lens)} tokens leaves no slot below max_len = {max_len}")
        self.d, self.page_size, self.dtype = d, page_size, dtype
        B, per = len(lens), -(-max_len // page_size)
        self.max_len = max_len
        order = torch.randperm(B * per, generator=torch.Generator().manual_seed(seed))
        self.table = order.view(B, per).to(torch.int32).to(device)
        self.lens = torch.tensor(lens, dtype=torch.int32, device=device)  # tokens held, the new one excluded
        self.layers = [Layer(d, seed * 1000 + i, device, dtype) for i in range(layers)]
        self.caches = [PagedCache(d, B * per, page_size, device, cache_dtype or dtype) for _ in range(layers)]
        half = d.head_dim // 2
        angle = torch.arange(max_len, device=device)[:, None] * d.rope_base ** (-torch.arange(half, device=device) / half)
        self.cos, self.sin = angle.cos(), angle.sin()

    def place(self) -> Place:
        """Of the new tokens, from the lengths on the device. A full sequence has no slot."""
        at = self.lens.long()
        page = (at // self.page_size).clamp_max(self.table.shape[1] - 1)
        slot = self.table.long().gather(1, page[:, None])[:, 0] * self.page_size + at % self.page_size
        held = (self.lens + 1).clamp_max(self.max_len)
        turn = at.clamp_max(self.max_len - 1)
        return Place(torch.where(at < self.max_len, slot, -1), held, self.cos[turn][:, None], self.sin[turn][:, None])

    def layer(self, i: int, x: torch.Tensor, residual: torch.Tensor | None, at: Place, trace: dict | None = None):
        """(x, residual) after layer i; ``trace``, if given, receives the steps' results."""
        from cb200 import ops

        d, w, cache = self.d, self.layers[i], self.caches[i]
        B, hd = x.shape[0], d.head_dim
        q8, s8, h = ops.add_rmsnorm_quant(x, w.norm_in, d.eps, residual, mode="fp8_block")
        h = x if h is None else h
        qkv = ops.fp8_block_gemm(q8, w.qkv[0], s8, w.qkv[1], out_dtype=self.dtype, bias=w.qkv_bias)
        heads = qkv.view(B, -1, hd)
        q, k = rope(heads[:, :d.heads + d.kv_heads], at).split([d.heads, d.kv_heads], dim=1)
        v = heads[:, d.heads + d.kv_heads:]
        ops.paged_kv_append(k, v, cache.k, cache.v, at.slots, cache.k_scale, cache.v_scale)
        attn = ops.paged_decode_attention(q, cache.k, cache.v, self.table, at.held, k_scale=cache.k_scale, v_scale=cache.v_scale)
        o = ops.fp8_block_gemm_dynamic(attn.view(B, -1), *w.o)
        q8m, s8m, h2 = ops.add_rmsnorm_quant(o, w.norm_mid, d.eps, h, mode="fp8_block")
        gate, up = ops.fp8_block_gemm(q8m, w.gate_up[0], s8m, w.gate_up[1], out_dtype=self.dtype).chunk(2, dim=-1)
        act = torch.nn.functional.silu(gate) * up
        out = ops.fp8_block_gemm_dynamic(act, *w.down)
        if trace is not None:
            trace.update(q8=q8, s8=s8, h=h, qkv=qkv, q=q, k=k, v=v, attn=attn, o=o, q8m=q8m, s8m=s8m, h2=h2, gate=gate, up=up,
                         act=act, out=out)
        return out, h2

    def step(self, x: torch.Tensor) -> torch.Tensor:
        """One new token per sequence: its hidden states [B, hidden] through all layers.
        The caches and ``lens`` then hold it."""
        residual, at = None, self.place()
        for i in range(len(self.layers)):
            x, residual = self.layer(i, x, residual, at)
        self.lens.add_((self.lens < self.max_len).to(torch.int32))
        return x + residual

    def step_bytes(self, tokens: int) -> int:
        """Weights, and keys and values of ``tokens`` tokens, that a step reads."""
        c = self.caches[0].k
        return sum(w.weight_bytes() for w in self.layers) + len(self.layers) * 2 * tokens * c.shape[2] * c.shape[3] * c.element_size()


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--batches", default="1,16,64")
    ap.add_argument("--context", type=int, default=4096)
    ap.add_argument("--layers", type=int, default=8)
    ap.add_argument("--page-size", type=int, default=64)
    ap.add_argument("--cache", default="bf16", choices=["bf16", "e4m3"])
    ap.add_argument("--steps", type=int, default=50)
    ap.add_argument("--out", default=None)
    a = ap.parse_args()
    from cb200 import ops

    dev, d, rows = torch.device("cuda"), Dims(), []
    with ClockSampler() as clocks:
        for B in (int(b) for b in a.batches.split(",")):
            # the timed steps leave the lengths where they are: the graph's own advance is taken back
            m = Decoder(d, a.layers, [a.context] * B, a.context + 64, a.page_size, dev, cache_dtype=FP8 if a.cache == "e4m3" else None)
            x = torch.randn(B, d.hidden, device=dev).to(torch.bfloat16)

            def step():
                m.step(x)
                m.lens.sub_(1)

            us = graph_time_us(step, inner=1, reps=a.steps)
            us_layer = us / a.layers
            read = m.step_bytes(B * (a.context + 1))
            r = {"batch": B, "context": a.context, "cache": a.cache, "layers": a.layers, "us_per_step": round(us, 1),
                 "us_per_layer": round(us_layer, 2), "tokens_per_s_64_layers": round(B / (us_layer * 64e-6)),
                 "read_gb": round(read / 1e9, 3), "read_tb_per_s": round(read / us / 1e6, 2)}
            rows.append(r)
            print(r, flush=True)
            if ops.device_status(dev) != 0:
                raise RuntimeError("a kernel recorded an error")
            del m
            torch.cuda.empty_cache()
    if a.out:
        save_json(a.out, {"experiment": "fp8_block_decode_layer", "gpu": gpu_info(), "dims": d.__dict__, "rows": rows,
                          "clocks": clocks.info})


if __name__ == "__main__":
    main()
