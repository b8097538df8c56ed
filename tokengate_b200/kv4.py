"""The 4-bit KV cache of one layer.

K and V rows of head_dim 128 as 4-bit codes with a bf16 step and a bf16 low per
group of 64 dims: 144 bytes per (slot, kv head) instead of the 512 of a bf16
cache. Written by ops.kv4_write (many rows) and ops.qk_norm_rope_append_kv4 (a
decode token), attended by ops.decode_attention_kv4, read back as bf16 by
ops.kv4_read. Slots are independent: writing one leaves the others untouched,
and a slot that was never written may hold anything (mask it).
"""
import torch

HEAD_DIM = 128
TILE_SLOTS = 32       # slots per tile of the cache's layout (csrc/kv4.cuh)
TILE_BYTES = 4608


class KV4Cache:
    """`capacity` slots of `batch` rows with `n_kv_heads` KV heads, on a CUDA device."""

    __slots__ = ("data", "batch", "capacity", "n_kv_heads", "bf16")

    def __init__(self, batch: int, capacity: int, n_kv_heads: int, device="cuda"):
        if batch < 1 or capacity < 1 or n_kv_heads < 1:
            raise ValueError(f"batch ({batch}), capacity ({capacity}) and n_kv_heads ({n_kv_heads}) must be positive")
        self.batch, self.capacity, self.n_kv_heads = int(batch), int(capacity), int(n_kv_heads)
        tiles = -(-self.capacity // TILE_SLOTS)
        self.data = torch.empty((self.batch, self.n_kv_heads, tiles, TILE_BYTES), dtype=torch.uint8, device=device)
        if not self.data.is_cuda:
            raise ValueError(f"a KV4Cache lives on a CUDA device (the B200 kernels have no CPU path), got {self.data.device}")
        self.bf16 = torch.empty(0, dtype=torch.bfloat16, device=self.data.device)   # makes the outputs (new_empty)

    # asked of the tensor at every call (0.1 us): a copied, unpickled or reassigned cache has its data elsewhere
    @property
    def ptr(self) -> int:
        return self.data.data_ptr()

    @property
    def index(self) -> int:
        return self.data.get_device()

    @property
    def device(self) -> torch.device:
        return self.data.device

    @property
    def nbytes(self) -> int:
        return self.data.numel()
