"""Paged KV cache: block tables, the HBM pool and the block allocator.

Drop-in for engine/model/kv_cache.py.  ``BlockTable`` and ``KVCacheManager`` are
host-side bookkeeping with the reference's exact semantics (FIFO free list with
``pop(0)``, kv_cache.py:150-227).  ``PhysicalKVCachePool`` keeps the reference's
layout ``[L, num_blocks, block_size, kv_heads, head_dim]`` for ``k_cache`` and
``v_cache`` (kv_cache.py:45-80) but allocates it in HBM in the model dtype.  The
decoder path writes and reads it only inside the CUDA kernels
(``b2_rope_kv_write``, ``b2_paged_attention``); ``store_kv``/``read_kv_sequence``
remain for API compatibility as device-side copies.

With ``KVCacheConfig.kv_dtype`` "int8" or "fp8_e4m3" the pool holds codes ``[L, num_blocks,
kv_heads, 16, head_dim]`` and a float32 scale per (layer, block, kv head); the kernels for it are
``b2_qk_norm_rope_kv_write_q8``, ``b2_paged_attention_q8``, ``b2_prefill_attention_q8`` and
``b2_kv_read_q8``.  ``DeviceBlockTables`` is the manager's bookkeeping kept on the GPU
(``b2_block_tables_extend``/``_truncate``) for steps that know their lengths there, such as
accepted drafts.
"""

from __future__ import annotations

import math
from typing import Dict, List, Optional, Sequence, Tuple, Union

import torch

from pythonintern_b200 import kernels
from pythonintern_b200.config import KVCacheConfig, ModelConfig
from pythonintern_b200.model.metadata import TokenMetadata
from pythonintern_b200._lib import cache_torch_dtype, torch_dtype


class BlockTable:
    """Logical token index -> (physical block, offset) for one sequence (kv_cache.py:13-43)."""

    def __init__(self, seq_id: str, block_size: int):
        self.seq_id = seq_id
        self.block_size = block_size
        self.physical_block_ids: List[int] = []
        self.num_tokens: int = 0

    def append_block(self, block_id: int):
        self.physical_block_ids.append(block_id)

    def num_allocated_blocks(self) -> int:
        return len(self.physical_block_ids)

    def get_physical_slot(self, logical_pos: int) -> Tuple[int, int]:
        block_idx = logical_pos // self.block_size
        offset = logical_pos % self.block_size
        assert block_idx < len(self.physical_block_ids), (
            f"sequence {self.seq_id}: token {logical_pos} falls in block {block_idx}, but only "
            f"{len(self.physical_block_ids)} blocks are allocated")
        return self.physical_block_ids[block_idx], offset


class PhysicalKVCachePool:
    """K/V pool ``[L, num_blocks, block_size, kv_heads, head_dim]`` in HBM (kv_cache.py:45-147).

    ``kv_dtype`` "int8" or "fp8_e4m3" stores 8-bit codes ``[L, num_blocks, kv_heads, 16, head_dim]``
    with ``k_scale``/``v_scale`` float32 ``[L, num_blocks, kv_heads]`` (None for the model's type);
    ``dtype`` stays the type of the values.
    """

    def __init__(self, num_blocks: int, block_size: int, num_local_kv_heads: int, head_dim: int,
                 num_layers: int, device="cuda", dtype=None, kv_dtype: str = "model"):
        self.num_blocks = num_blocks
        self.block_size = block_size
        self.num_local_kv_heads = num_local_kv_heads
        self.head_dim = head_dim
        self.num_layers = num_layers
        self.device = torch.device(device)
        if self.device.type not in ("cuda", "meta"):
            # "meta" gives a shape-only pool for host-side bookkeeping without a GPU.
            raise ValueError("PhysicalKVCachePool lives in HBM: device must be cuda")
        dt = torch_dtype(dtype)
        self.kv_dtype = kv_dtype
        self.value_dtype = dt
        self.k_scale: Optional[torch.Tensor] = None
        self.v_scale: Optional[torch.Tensor] = None
        if kv_dtype == "model":
            shape = (num_layers, num_blocks, block_size, num_local_kv_heads, head_dim)
        else:
            dt = cache_torch_dtype(kv_dtype)
            if block_size != 16 or head_dim not in (32, 64, 128):
                raise ValueError(f"a KV pool of {kv_dtype} has blocks of 16 tokens and heads of 32, 64 or 128; "
                                 f"got block_size {block_size}, head_dim {head_dim}")
            shape = (num_layers, num_blocks, num_local_kv_heads, block_size, head_dim)
            scales = (num_layers, num_blocks, num_local_kv_heads)
            self.k_scale = torch.zeros(scales, dtype=torch.float32, device=self.device)
            self.v_scale = torch.zeros(scales, dtype=torch.float32, device=self.device)
        self.k_cache = torch.zeros(shape, dtype=dt, device=self.device)
        self.v_cache = torch.zeros(shape, dtype=dt, device=self.device)

    @property
    def dtype(self) -> torch.dtype:
        return self.value_dtype

    @property
    def quantised(self) -> bool:
        return self.k_scale is not None

    def _refuse_store(self):
        if self.quantised:
            raise ValueError(f"a KV pool of {self.kv_dtype} is written by the attention kernels only: a block's "
                             "tokens share a scale")

    def store_kv(self, layer_idx: int, physical_block_id: int, offset: int, k: torch.Tensor, v: torch.Tensor):
        """One token's K/V ``[kv_heads, head_dim]`` into a slot (kv_cache.py:85-100)."""
        self._refuse_store()
        self.k_cache[layer_idx, physical_block_id, offset].copy_(k)
        self.v_cache[layer_idx, physical_block_id, offset].copy_(v)

    def store_kv_batch(self, layer_idx: int, block_ids: List[int], offsets: List[int], k: torch.Tensor,
                       v: torch.Tensor):
        """Tokens ``i`` into slots ``(block_ids[i], offsets[i])`` (kv_cache.py:102-119)."""
        self._refuse_store()
        b = torch.as_tensor(block_ids, dtype=torch.long, device=self.device)
        o = torch.as_tensor(offsets, dtype=torch.long, device=self.device)
        self.k_cache[layer_idx, b, o] = k.to(self.k_cache.dtype)
        self.v_cache[layer_idx, b, o] = v.to(self.v_cache.dtype)

    def read_kv_sequence(self, layer_idx: int, block_ids: List[int], seq_len: int):
        """Gather a sequence's first ``seq_len`` K/V rows (kv_cache.py:121-147)."""
        if not block_ids:
            e = torch.empty((0, self.num_local_kv_heads, self.head_dim), dtype=self.dtype, device=self.device)
            return e, e.clone()
        if self.quantised:
            ids = torch.as_tensor(block_ids, dtype=torch.int32, device=self.device)
            k, v = kernels.kv_read_q8(self.k_cache, self.v_cache, self.k_scale, self.v_scale, layer_idx, ids, self.dtype)
            return k.flatten(0, 1)[:seq_len], v.flatten(0, 1)[:seq_len]
        idx = torch.as_tensor(block_ids, dtype=torch.long, device=self.device)
        k = self.k_cache[layer_idx].index_select(0, idx).view(-1, self.num_local_kv_heads, self.head_dim)
        v = self.v_cache[layer_idx].index_select(0, idx).view(-1, self.num_local_kv_heads, self.head_dim)
        return k[:seq_len], v[:seq_len]


class KVCacheManager:
    """Block allocation, freeing and per-sequence tables (kv_cache.py:150-227)."""

    def __init__(self, config: KVCacheConfig, model_config: ModelConfig, world_size: int):
        self.config = config
        self.block_size = config.block_size
        self.total_blocks = config.num_blocks
        self.free_blocks: List[int] = list(range(config.num_blocks))
        self.block_tables: Dict[str, BlockTable] = {}
        num_local_kv_heads = max(1, model_config.num_kv_heads // world_size)
        device = config.device if config.device not in ("cpu", None) else "cuda"
        group = model_config.num_queries_per_kv
        if config.kv_dtype != "model" and group > 16:
            raise ValueError(f"a KV pool of {config.kv_dtype} serves up to 16 q heads to a kv head; the model has {group}")
        self.pool = PhysicalKVCachePool(
            num_blocks=config.num_blocks, block_size=config.block_size, num_local_kv_heads=num_local_kv_heads,
            head_dim=model_config.head_dim, num_layers=model_config.num_layers, device=device,
            dtype=model_config.dtype, kv_dtype=config.kv_dtype)

    @property
    def free_block_count(self) -> int:
        return len(self.free_blocks)

    @property
    def allocated_block_count(self) -> int:
        return self.total_blocks - len(self.free_blocks)

    def allocate_blocks_for_sequence(self, seq_id: str, num_tokens: int) -> BlockTable:
        needed_blocks = math.ceil(num_tokens / self.block_size)
        if needed_blocks > len(self.free_blocks):
            raise MemoryError(f"sequence {seq_id} needs {needed_blocks} KV blocks; "
                              f"{len(self.free_blocks)} are free")
        if seq_id not in self.block_tables:
            self.block_tables[seq_id] = BlockTable(seq_id, self.block_size)
        table = self.block_tables[seq_id]
        for _ in range(needed_blocks - len(table.physical_block_ids)):
            table.append_block(self.free_blocks.pop(0))
        table.num_tokens = num_tokens
        return table

    def append_token(self, seq_id: str) -> Tuple[int, int]:
        table = self.block_tables[seq_id]
        new_token_pos = table.num_tokens
        block_idx = new_token_pos // self.block_size
        offset = new_token_pos % self.block_size
        if block_idx >= len(table.physical_block_ids):
            if not self.free_blocks:
                raise MemoryError(f"KV pool exhausted: no free block for the next token of sequence {seq_id}")
            table.append_block(self.free_blocks.pop(0))
        table.num_tokens += 1
        return table.physical_block_ids[block_idx], offset

    def free_sequence(self, seq_id: str) -> int:
        if seq_id not in self.block_tables:
            return 0
        table = self.block_tables.pop(seq_id)
        self.free_blocks.extend(table.physical_block_ids)
        return len(table.physical_block_ids)


class DeviceBlockTables:
    """``KVCacheManager``'s bookkeeping on the GPU: tables, lengths and the FIFO free list.

    A fixed number of sequence slots (rows).  ``extend`` takes the blocks of a step's new tokens and
    returns the step's ``TokenMetadata``; ``truncate`` gives blocks back (rejected drafts; 0 frees a
    slot).  Blocks go out and come back in the order of ``KVCacheManager`` serving the rows in turn.
    Nothing comes back to the host: a step that cannot be served (too few free blocks, a row past its
    width) changes nothing here, becomes a step without tokens, and is reported by
    ``_lib.check_device_status`` (``MemoryError``, ``IndexError``).
    """

    def __init__(self, n_seqs: int, max_blocks_per_seq: int, num_blocks: int, block_size: int = 16, device="cuda"):
        dev = torch.device(device)
        if dev.type == "cuda" and dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        self.device = dev
        self.n_seqs = n_seqs
        self.block_size = block_size
        self.tables = torch.full((n_seqs, max_blocks_per_seq), -1, dtype=torch.int32, device=dev)
        self.lens = torch.zeros(n_seqs, dtype=torch.int32, device=dev)
        self.free_ring = torch.arange(num_blocks, dtype=torch.int32, device=dev)
        self.free_state = torch.tensor([0, num_blocks, 0, 0], dtype=torch.int32, device=dev)

    def _lengths(self, x: Union[Sequence[int], torch.Tensor]) -> torch.Tensor:
        if not isinstance(x, torch.Tensor):
            x = torch.tensor(x, dtype=torch.int32).to(self.device)
        if x.shape != (self.n_seqs,) or x.dtype != torch.int32 or x.device != self.device:
            raise ValueError(f"one int32 length per sequence slot ({self.n_seqs}) on {self.device}; "
                             f"got {x.dtype} {tuple(x.shape)} on {x.device}")
        return x.contiguous()

    def extend(self, new_lens: Union[Sequence[int], torch.Tensor], n_tokens: Optional[int] = None) -> TokenMetadata:
        """Metadata of one call over ``new_lens[s]`` new tokens of every slot ``s`` behind those it holds.

        ``new_lens`` on the device needs ``n_tokens``, its sum, as shapes are the host's to know.
        ``last_rows`` is 0 for a slot without new tokens: its sampled token means nothing.
        """
        if n_tokens is None:
            if isinstance(new_lens, torch.Tensor):
                raise ValueError("new_lens on the device needs n_tokens")
            n_tokens = int(sum(new_lens))
        if n_tokens < 1:
            raise ValueError("a step needs at least one new token")
        new = self._lengths(new_lens)
        n = self.n_seqs
        ctx0 = self.lens.clone()
        m = kernels.block_tables_extend(self.tables, self.lens, new, n_tokens, self.block_size, self.free_ring,
                                        self.free_state)
        return TokenMetadata(n_tokens=n_tokens, is_prefill=True, rope_pos=m.positions, store_pos=m.positions,
                             table_index=m.table_index, tables=self.tables, ctx_lens=m.ctx_lens,
                             max_ctx=self.tables.shape[1] * self.block_size, compat_pad=False,
                             seq_start=m.seq_start, n_seqs=n, seq_ctx0=ctx0, last_rows=m.last_rows.clamp_(min=0))

    def truncate(self, keep_lens: Union[Sequence[int], torch.Tensor]):
        """Every slot keeps its first ``keep_lens[s]`` tokens; the blocks behind them are free again."""
        kernels.block_tables_truncate(self.tables, self.lens, self._lengths(keep_lens), self.block_size,
                                      self.free_ring, self.free_state)
