"""Engine options.  Names and defaults are the reference's server config keys
(internal/config/config.go:33-78): max_batch_size 64, max_token_budget 4096,
max_queue_depth 256, prefill_chunk_size 512, block_size 16, max_memory_fraction 0.9."""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional


@dataclass
class EngineConfig:
    dtype: str = "bfloat16"                # "bfloat16" (serving kernels) | "float32" (true 32-bit)
    block_size: int = 16                   # tokens per cache page
    num_blocks: Optional[int] = None       # pages per cache group; None => from max_memory_fraction
    max_memory_fraction: float = 0.9
    max_batch_size: int = 64               # sequences per step
    max_token_budget: int = 4096           # tokens per step
    max_queue_depth: int = 256
    prefill_chunk_size: int = 512          # most prompt tokens of one request per step; 0 = no cut
    max_model_len: Optional[int] = None    # longest sequence; None => max_position_embeddings
    strict_fcfs: bool = True               # the head of the queue blocks those behind it; False: a
                                           # request that does not fit is passed over, as in the
                                           # reference (internal/scheduler/fcfs.go:130-161)
    cache_bits: Optional[int] = None       # 4 or 8: keys and values are held in so many bits (gollmgo_b200/cache/packed.py);
                                           # None: in dtype
    cuda_graphs: bool = True               # capture decode-only steps
    capture_at_start: bool = True          # capture every batch bucket when the engine is built, not at first use
    state_slots: Optional[int] = None      # requests that can be admitted at once (each holds a state slot);
                                           # None => twice max_batch_size, at least 8
    device: int = 0

    def validate(self) -> None:
        if self.dtype not in ("bfloat16", "float32"):
            raise ValueError(f"dtype must be bfloat16 or float32, got {self.dtype!r}")
        if self.block_size <= 0 or self.block_size & (self.block_size - 1):
            raise ValueError(f"block_size must be a power of two, got {self.block_size}")
        if self.cache_bits not in (None, 4, 8):
            raise ValueError(f"cache_bits must be 4, 8 or None, got {self.cache_bits!r}")
        if self.cache_bits and not 4 <= self.block_size <= 256:
            raise ValueError(f"a packed cache has pages of 4 to 256 tokens, got block_size {self.block_size}")
        if self.max_batch_size <= 0:
            raise ValueError("max_batch_size must be positive")
        if self.max_token_budget <= 0:
            raise ValueError("max_token_budget must be positive")
        if not (0.0 < self.max_memory_fraction <= 1.0):
            raise ValueError("max_memory_fraction must be in (0, 1]")
        if self.state_slots is not None and self.state_slots <= 0:
            raise ValueError("state_slots must be positive")
        if self.prefill_chunk_size < 0:
            raise ValueError("prefill_chunk_size must be >= 0")
