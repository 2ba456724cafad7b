"""Block tables of a fixed batch of sequences that live on the GPU.

PagedKVCache.prepare_step builds a step's metadata on the host from Python
tables and copies it over.  For a batch that is decoded together (a fixed set of
prompts, all generating), DeviceStepTables keeps the tables, the lengths and the
free list in device memory instead, and ops.build_step_tables derives each step
from the request lengths in one launch: a decode step copies nothing to the
device.  The metadata is what forward_layer / forward_layer_qkv take (call them
with advance=False: the lengths are kept here, not in the cache).

The host follows the lengths and the number of free blocks (both follow from the
lengths it asks for), so a step that the free list is too short for raises
OutOfBlocks before anything is launched; the block ids stay on the device until
`release` gives all of them back.  Reference: the table growth of
mini_engine/scheduler.py:79-156.
"""

from __future__ import annotations

import torch

from . import ops
from .block_manager import BlockManager, OutOfBlocks, StepMetadata


class DeviceStepTables:
    """n_seqs sequences of up to max_blocks_per_seq blocks, over `blocks` blocks
    taken from the manager (OutOfBlocks, and none taken, if it has fewer)."""

    def __init__(self, mgr: BlockManager, n_seqs: int, max_blocks_per_seq: int, blocks: int):
        if mgr.device is None:
            raise RuntimeError("pagedkv: DeviceStepTables needs a manager with pools on a GPU")
        if n_seqs <= 0 or max_blocks_per_seq <= 0 or blocks <= 0:
            raise ValueError("pagedkv: n_seqs, max_blocks_per_seq and blocks must be positive")
        if mgr.num_free < blocks:
            raise OutOfBlocks()
        self.mgr, self.n_seqs, self.width = mgr, n_seqs, max_blocks_per_seq
        self.blocks = [mgr.allocate() for _ in range(blocks)]
        dev = mgr.device
        # the first one allocated is the first one taken (from the end)
        self.free_blocks = torch.tensor(self.blocks[::-1], dtype=torch.int32).to(dev)
        self.n_free = torch.full((1,), blocks, dtype=torch.int32, device=dev)
        self.tables = torch.zeros((n_seqs, max_blocks_per_seq), dtype=torch.int32, device=dev)
        self.lens_dev = torch.zeros(n_seqs, dtype=torch.int32, device=dev)
        self._ones = torch.ones(n_seqs, dtype=torch.int32, device=dev)
        self.lens = [0] * n_seqs
        self.left = blocks
        self.positions: torch.Tensor | None = None  # int64 [n_tokens] of the last step

    def step(self, num_new: list[int]) -> StepMetadata:
        """The metadata of a step that gives sequence i num_new[i] more tokens,
        laid out as prepare_step's (sequences in order).  The tokens' positions
        are in `positions`."""
        if self.blocks is None:
            raise RuntimeError("pagedkv: the tables were released")
        if len(num_new) != self.n_seqs or any(n < 0 for n in num_new):
            raise ValueError(f"pagedkv: num_new must hold {self.n_seqs} token counts")
        bs = self.mgr.block_size
        totals = [p + n for p, n in zip(self.lens, num_new)]
        if max(totals) > self.width * bs:
            raise ValueError(f"pagedkv: {max(totals)} tokens, but a table holds {self.width * bs}")
        need = sum(-(-t // bs) - -(-p // bs) for t, p in zip(totals, self.lens))
        if need > self.left:
            raise OutOfBlocks()
        self.mgr.flush_copies()
        nd = 0
        while nd < self.n_seqs and num_new[nd] == 1:
            nd += 1
        new_dev = self._ones
        if nd < self.n_seqs:
            new_dev = torch.tensor(num_new, dtype=torch.int32).pin_memory().to(self.mgr.device, non_blocking=True)
        T = sum(num_new)
        prior = self.lens_dev
        st = ops.build_step_tables(self.tables, self.free_blocks, self.n_free, prior, new_dev, bs, T, err=self.mgr.err)
        meta = StepMetadata(
            # no sequence of a cache has such an id: its lengths stay as they are even
            # if a layer is told to advance them
            seq_ids=[-1 - i for i in range(self.n_seqs)], num_new=list(num_new), num_prior=self.lens, n_tokens=T,
            n_decode=nd, max_query_len=max(num_new[nd:], default=0), slot_mapping=st.slot_mapping,
            block_tables=self.tables, context_lens=st.context_lens,
            # relative to the rows behind the decode sequences' one each
            query_start_loc=st.query_start_loc[nd:] - nd if nd else st.query_start_loc,
            num_prior_dev=prior)
        self.lens_dev, self.n_free, self.positions = st.context_lens, st.n_free, st.positions
        self.lens, self.left = totals, self.left - need
        return meta

    def release(self) -> None:
        """Give every block back to the manager."""
        if self.blocks is not None:
            for b in self.blocks:
                self.mgr.decref(b)
            self.blocks = None
