"""A dense KV cache in eight bits: every token's rows as e4m3 codes with a scale a block of rows and KV head (``ops.Fp8KVCache``), all of them attended
to (``ops.Fp8Attention``).  Half the bytes of a bf16 cache, and of what a decode step reads.  The methods a decode loop calls are those of
``polar_cache`` (no counterpart in the reference, whose caches are bf16)."""
from __future__ import annotations

import torch

from .. import ops
from .cache import KV_Cache


class fp8_cache(KV_Cache):
    """``max_length`` rows a sequence, for the prompt and what follows; every sequence has as many.  ``block``: rows to a scale.  For one stream at a time,
    and not for a captured graph: lengths are numbers of the moment of the call."""

    def __init__(self, valid_start, layer_num: int, batch_size: int, max_length: int, num_key_value_heads: int, num_heads: int, head_dim: int,
                 dtype: torch.dtype, layer_mapping: dict, num_gpus: int = 1, model_size: int = 0, block: int = 64) -> None:
        super().__init__(layer_num, batch_size, max_length, num_key_value_heads, num_heads, head_dim, dtype, layer_mapping, num_gpus, model_size)
        if head_dim != ops.HEAD_DIM:
            raise ValueError("head_dim must be 128")
        if dtype not in (torch.bfloat16, torch.float32):
            raise ValueError("dtype must be bfloat16 or float32")
        if num_heads % num_key_value_heads:
            raise ValueError("num_heads must be a multiple of num_key_value_heads")
        self.valid_start = valid_start
        self.group_size = num_heads // num_key_value_heads
        self.device = torch.device(list(layer_mapping.values())[0] if layer_mapping else "cuda:0")
        if self.device.type != "cuda":
            raise RuntimeError("GPU required")
        self.layers = [ops.Fp8KVCache(batch_size, num_key_value_heads, max_length, self.device, block) for _ in range(layer_num)]
        self.max_tokens = min(1024, 8192 // self.group_size)  # a call of compute
        self._attention = ops.Fp8Attention(batch_size, num_key_value_heads, self.group_size, self.max_tokens, max_length, self.device)
        self.current_seq_len = [0] * layer_num
        self._prefilled = [[0] * batch_size for _ in range(layer_num)]

    def _start_of(self, batch_idx: int) -> int:
        vs = self.valid_start
        return int(vs[batch_idx]) if hasattr(vs, "__len__") else int(vs)

    def prefill_update_kv_cache(self, query_states, key_states, value_states, layer_idx, batch_idx):
        """A prompt's rows [bsz,S,Hkv,D] from valid_start on: of sample ``batch_idx`` (bsz 1), or of all (bsz = batch_size, batch_idx 0).  They replace what
        the cache held; all samples' prompts have as many rows.  Returns the states from valid_start on."""
        bsz, seq_len = key_states.shape[:2]
        if bsz not in (1, self.batch_size):
            raise RuntimeError(f"one sample, or all {self.batch_size} of the cache")
        b0 = int(batch_idx) if bsz == 1 else 0
        if not 0 <= b0 < self.batch_size:
            raise RuntimeError("no such sample")
        vs = self._start_of(b0)
        if any(self._start_of(b) != vs for b in range(b0, b0 + bsz)):
            raise RuntimeError("samples stored by one call have one valid_start")
        k, v = key_states[:, vs:], value_states[:, vs:]
        n = k.shape[1]
        if n < 1 or n > self.max_length:
            raise RuntimeError(f"a prompt of {n} rows in a cache of {self.max_length}")
        if bsz != 1 and batch_idx != 0:
            return k, v
        cache = self.layers[layer_idx]
        if bsz != self.batch_size:
            cache = ops.Fp8KVCache.from_codes(*(t[b0:b0 + 1] for t in (cache.k, cache.k_scale, cache.v, cache.v_scale)), block=cache.block)
        cache.store(k, v)
        done = self._prefilled[layer_idx]
        done[b0:b0 + bsz] = [n] * bsz
        self.current_seq_len[layer_idx] = n
        if layer_idx == self.layer_num - 1 and b0 + bsz == self.batch_size:
            self.context = n
        return k, v

    def _rows_of(self, layer_idx):
        """How many rows every sequence has in a layer."""
        n, rows = self.current_seq_len[layer_idx], self._prefilled[layer_idx]
        if rows.count(n) != self.batch_size:
            raise RuntimeError("sequences of several lengths: every sample's prompt has to have as many rows")
        return n

    def decode_update_kv_cache(self, key_states, value_states, layer_idx):
        """Rows [bs,T,Hkv,D] of the next tokens of every sequence, behind those that are there."""
        n, T = self._rows_of(layer_idx), key_states.shape[1]
        if n + T > self.max_length:
            raise RuntimeError(f"{n} + {T} rows in a cache of {self.max_length}")
        self.layers[layer_idx].store(key_states, value_states, n)
        self.current_seq_len[layer_idx] = n + T
        self._prefilled[layer_idx] = [n + T] * self.batch_size
        if layer_idx == 0:
            self.context += T
        return None, None

    def compute(self, queries, layer_idx):
        """Attention of the last T tokens, [bs,T,Hq,D] -> [bs,T,Hq,D]: each sees the rows up to its own."""
        return self._attention.run(queries, self.layers[layer_idx], [(0, self._rows_of(layer_idx))])

    def draft_attend(self, queries, key_states, value_states, layer_idx, mask=None):
        raise RuntimeError("drafted tokens: polar_cache attends to them")

    def sync(self, layer_idx, batch_idx):
        """Nothing to wait for."""
