"""A key-value cache in pages for sequences of different lengths, which Transformer.prefill and generate_ragged fill and
read: the reference decodes all sequences of a batch at one position over a dictionary of (B, H, S, hd) tensors
(smlm/model.py:97-105)."""
import torch

from . import kernels


class PagedLayer:
    """One attention layer's pages, and the plan of the pass that is running (shared by all layers)."""

    def __init__(self, cache, pages):
        self.cache, self.pages = cache, pages

    @property
    def plan(self):
        return self.cache.plan


class PromptPlan:
    """Tokens of several sequences in a row: their positions and slots, where each sequence's begin, and, where some follow
    cached ones, the slots of all keys and where each sequence's of these begin."""

    def __init__(self, positions, slots, cu_q, all_slots=None, cu_k=None):
        self.positions, self.slots, self.cu_q, self.all_slots, self.cu_k = positions, slots, cu_q, all_slots, cu_k


class StepPlan:
    """One token for every sequence: `lengths` (B,) int32 with it."""

    def __init__(self, positions, slots, block_table, lengths):
        self.positions, self.slots, self.block_table, self.lengths = positions, slots, block_table, lengths


class PagedKVCache:
    """n_seqs sequences of up to max_len tokens each in pages of page_size tokens, every layer's in bf16 or 4 bits (kind "bf16",
    "q4").  num_pages pages are shared by all sequences (by default enough for all at full length); a sequence gets more as
    it grows and gives them back with clear().  The host keeps the lengths; block_table and lengths are on the device,
    where a captured decode step reads them."""

    @torch.inference_mode(False)                       # later calls, outside of it, write what is made here
    def __init__(self, n_layers, n_seqs, max_len, n_kv_heads, head_dim, page_size=64, kind="bf16", num_pages=None, device="cuda"):
        if n_seqs < 1 or max_len < 1 or page_size < 1:
            raise ValueError(f"PagedKVCache: {n_seqs} sequences of {max_len} tokens in pages of {page_size}")
        per_seq = -(-max_len // page_size)
        num_pages = n_seqs * per_seq if num_pages is None else num_pages
        self.n_seqs, self.max_len, self.page_size, self.kind, self.num_pages = n_seqs, max_len, page_size, kind, num_pages
        self.n_kv_heads, self.head_dim = n_kv_heads, head_dim
        self.layers = [PagedLayer(self, kernels.kv_pages(num_pages, n_kv_heads, page_size, head_dim, kind, device))
                       for _ in range(n_layers)]
        self.block_table = torch.full((n_seqs, per_seq), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(n_seqs, dtype=torch.int32, device=device)
        self.seq_lens = [0] * n_seqs                   # the lengths, on the host
        self._pages = [[] for _ in range(n_seqs)]
        self._free = list(range(num_pages - 1, -1, -1))
        self.plan = None
        self.decoding = {}                             # Transformer.generate_ragged's buffers and graph

    @property
    def device(self):
        return self.block_table.device

    def clear(self, seq=None):
        """Forgets one sequence, or all of them; its pages are free again."""
        for b in range(self.n_seqs) if seq is None else [seq]:
            self._free += self._pages[b]
            self._pages[b] = []
            self.seq_lens[b] = 0
        self.refresh()

    def reserve(self, new):
        """Pages for new[b] more tokens of every sequence; ValueError, with nothing changed, where they do not fit."""
        if len(new) != self.n_seqs or any(n < 0 for n in new):
            raise ValueError(f"PagedKVCache: expected {self.n_seqs} counts of new tokens, got {new}")
        need = []
        for b, n in enumerate(new):
            if self.seq_lens[b] + n > self.max_len:
                raise ValueError(f"PagedKVCache: sequence {b} has {self.seq_lens[b]} tokens, {n} more exceed {self.max_len}")
            need.append(max(0, -(-(self.seq_lens[b] + n) // self.page_size) - len(self._pages[b])))
        if sum(need) > len(self._free):
            raise ValueError(f"PagedKVCache: {sum(need)} pages of {self.page_size} tokens are needed, {len(self._free)} are free")
        for b, n in enumerate(need):
            for _ in range(n):
                self._pages[b].append(self._free.pop())
        self.refresh()

    def refresh(self):
        """The device's block table and lengths as the host has them."""
        rows = [p + [-1] * (self.block_table.shape[1] - len(p)) for p in self._pages]
        self.block_table.copy_(torch.tensor(rows, dtype=torch.int32))
        self.lengths.copy_(torch.tensor(self.seq_lens, dtype=torch.int32))

    def _slots(self, b, first, end):
        t = torch.arange(first, end)
        return torch.tensor(self._pages[b] + [0], dtype=torch.int64)[t // self.page_size] * self.page_size + t % self.page_size

    def plan_prompts(self, new):
        """The plan of a pass over new[b] more tokens of each sequence, which have pages (reserve); the lengths grow by them
        (advance) behind the pass."""
        at = lambda parts: torch.cat(parts).to(self.device)  # noqa: E731
        cu = lambda counts: torch.tensor([0] + counts).cumsum(0).to(self.device, torch.int32)  # noqa: E731
        ends = [n + m for n, m in zip(self.seq_lens, new)]
        positions = at([torch.arange(n, e) for n, e in zip(self.seq_lens, ends)])
        slots = at([self._slots(b, n, e) for b, (n, e) in enumerate(zip(self.seq_lens, ends))])
        if not any(n and m for n, m in zip(self.seq_lens, new)):
            return PromptPlan(positions, slots, cu(list(new)))
        whole = [e if m else 0 for e, m in zip(ends, new)]        # what the pass attends to
        return PromptPlan(positions, slots, cu(list(new)), at([self._slots(b, 0, e) for b, e in enumerate(whole)]), cu(whole))

    def plan_step(self):
        """The plan of a pass over one more token of every sequence, from the device's lengths (which a captured step advances)."""
        if self.lengths.is_cuda:
            positions, slots, lengths = kernels.paged_step(self.block_table, self.lengths, self.page_size, self.max_len)
            return StepPlan(positions, slots, self.block_table, lengths)
        pos = self.lengths.long()
        page = self.block_table.gather(1, (pos // self.page_size).clamp_(max=self.block_table.shape[1] - 1).unsqueeze(1)).squeeze(1)
        # a sequence at its end has no slot: nothing is written
        slots = torch.where((page >= 0) & (pos < self.max_len), page.long() * self.page_size + pos % self.page_size, -1)
        return StepPlan(pos, slots, self.block_table, self.lengths + 1)

    def advance(self, new):
        """new[b] more tokens of each sequence are in the pages."""
        self.seq_lens = [n + m for n, m in zip(self.seq_lens, new)]
        self.lengths.copy_(torch.tensor(self.seq_lens, dtype=torch.int32))
