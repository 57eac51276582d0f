"""Speculative decoding with drafted token trees: one forward over every request's tree instead of one per token.

A step takes, per request, the tokens a drafter proposes as a tree below the last accepted token, runs the model over all of them at once and
keeps the longest path the model itself would have produced greedily, plus the token behind it: between one and depth + 1 tokens per request and
forward, those of greedy decoding whatever was drafted.  (Up to the rounding of the logits: plain decoding has products of other shapes and another
order of sums, and two tokens within that of each other may change places.)  Everything between the drafts and the accepted tokens happens on the
device (``ops.prepare_extend`` -> model -> ``ops.argmax`` -> ``ops.accept_tree``, with ``ops.token_logprobs`` where they are asked for), in one captured
hipGraph per decoder.  The reference decodes one token per step (mini_sglang/managers/scheduler.py:409-419) and has no counterpart.

Slots that rejected drafts leave behind stay with their request and are used by its next step; ``sync_host`` gives them back to the page allocator.
"""
from __future__ import annotations

from typing import List, Optional, Sequence, Tuple

import torch

from .. import ops
from .batch_info import BatchInfo, ForwardMode

_REFUSED = {1: "free list exhausted", 2: "context longer than the page table row", 3: "inconsistent lengths", 4: "more drafted nodes than announced"}


class TreeDecoder:
    """``max_nodes``: most nodes of a request's tree, the root (its last token) included.  ``max_new_tokens``: how far the contexts may grow
    before the captured bounds have to be renewed (done when needed).  ``logprobs``: None, or the number of alternatives to report with every
    accepted token's log probability (``last_logprobs``).  The step is captured inside torch's inference mode, like this package's other captured
    loops: as long as such a graph was the first one alive in the process, torch refuses captures outside inference mode."""

    def __init__(self, model_runner, batch: BatchInfo, max_nodes: int, *, max_new_tokens: int = 1024, logprobs: Optional[int] = None,
                 use_graph: bool = True):
        mr = model_runner
        if not 1 <= max_nodes <= 64 * ops.TREE_MAX_WORDS:
            raise ValueError(f"max_nodes {max_nodes} outside 1..{64 * ops.TREE_MAX_WORDS}")
        if any(r.sampling_params.temperature != 0 for r in batch.reqs):
            raise ValueError("drafted trees are accepted greedily: temperature must be 0")
        self.mr, self.batch, self.max_nodes, self.max_new_tokens, self.logprobs = mr, batch, max_nodes, max_new_tokens, logprobs
        self.use_graph, self.vocab = use_graph, mr.model_config.vocab_size
        self.bs, dev = batch.batch_size, mr.device
        bs, rows = self.bs, self.bs * max_nodes
        i32 = dict(dtype=torch.int32, device=dev)
        self.req_pool_indices = batch.req_pool_indices.to(**i32).clone()
        self.prefix_lens = batch.seq_lens.to(**i32).clone()     # tokens in the cache
        self.alloc_lens = self.prefix_lens.clone()              # positions with a table entry
        self.new_lens = torch.zeros(bs, **i32)
        self.input_ids, self.parents = torch.zeros(rows, **i32), torch.zeros(rows, **i32)
        self.positions, self.out_cache_loc = torch.zeros(rows, **i32), torch.zeros(rows, **i32)
        self.tree_mask = torch.zeros((rows, -(-max_nodes // 64)), dtype=torch.int64, device=dev)
        self.cu_seqlens_q, self.seq_lens = torch.zeros(bs + 1, **i32), torch.zeros(bs, **i32)
        self.status = torch.zeros(1, **i32)
        self.free_pages, self.free_range = torch.zeros(mr.page_allocator.page_num, **i32), torch.zeros(2, **i32)
        self.accept_lens, self.next_tokens = torch.zeros(bs, **i32), torch.zeros(bs, **i32)
        self.accept_rows, self.accept_tokens = torch.zeros((bs, max_nodes), **i32), torch.zeros((bs, max_nodes), **i32)
        self.layers = ops.kv_layers(mr.kv_cache_pool.k_buffer, mr.kv_cache_pool.v_buffer)
        self.seq_lens_cpu = batch.seq_lens_cpu.clone()
        self.synced_lens = self.seq_lens_cpu.clone()            # the batch's lengths as this decoder last took or left them
        self.reqs = list(batch.reqs)
        self.ahead = [len(r.token_ids) - int(n) for r, n in zip(self.reqs, self.seq_lens_cpu)]  # tokens a request has beyond its cached ones
        self.last_logprobs: List[list] = [[] for _ in range(bs)]
        self._scores = None
        self._upload_free_list()
        self._prepare()

    # ------------------------------------------------------------------ set-up
    def _upload_free_list(self) -> None:
        fp = self.mr.page_allocator.free_page
        self.free_pages[: fp.numel()].copy_(fp)
        self.free_range.copy_(torch.tensor([0, fp.numel()], dtype=torch.int32))
        self._uploaded, self.pending = fp.clone(), 0

    def _host_pages_changed(self) -> bool:
        changed = not torch.equal(self._uploaded, self.mr.page_allocator.free_page)
        if changed and self.pending:
            raise RuntimeError("the page allocator changed under a running TreeDecoder: call sync_host() before other batches allocate or free")
        return changed

    def _take_lengths(self) -> None:
        """The batch's lengths, where its requests were decoded by other means since the last sync_host()."""
        b = self.batch
        if len(b.reqs) != self.bs or any(r is not mine for r, mine in zip(b.reqs, self.reqs)):
            raise RuntimeError("the batch's requests changed: a TreeDecoder serves those it was made for")
        if not torch.equal(b.seq_lens_cpu, self.synced_lens):
            if self.pending:
                raise RuntimeError("the batch was decoded by other means under a running TreeDecoder: call sync_host() before")
            self.prefix_lens.copy_(b.seq_lens)
            self.alloc_lens.copy_(self.prefix_lens)
            self.seq_lens_cpu, self.synced_lens = b.seq_lens_cpu.clone(), b.seq_lens_cpu.clone()
        if any(len(r.token_ids) - n != a for r, n, a in zip(self.reqs, self.seq_lens_cpu.tolist(), self.ahead)):
            raise RuntimeError("a request's tokens and its cached positions do not go together any more")

    def _prepare(self) -> None:
        """Bounds, metadata and (captured) step for contexts up to max_new_tokens longer than now."""
        mr = self.mr
        # no longer than a page table row: prepare_extend refuses a step that would outgrow it
        self.bound = min(int(self.seq_lens_cpu.max()) + self.max_new_tokens + self.max_nodes, mr.req_to_token_pool.req_to_token.shape[1])
        self.static_batch = BatchInfo(
            forward_mode=ForwardMode.VERIFY, input_ids=self.input_ids, positions=self.positions, seq_lens=self.seq_lens,
            prefix_seq_lens=self.prefix_lens, input_seq_lens_max=self.max_nodes, max_seq_len=self.bound,
            total_kv=int(self.seq_lens_cpu.sum()) + self.bs * (self.max_nodes + self.max_new_tokens // 2), cu_seqlens_q=self.cu_seqlens_q,
            tree_mask=self.tree_mask, out_cache_loc=self.out_cache_loc, req_pool_indices=self.req_pool_indices,
            req_to_token_pool=mr.req_to_token_pool, kv_cache_pool=mr.kv_cache_pool, page_allocator=mr.page_allocator, attn_backend=mr.attn_backend,
            reqs=[], device=mr.device)
        mr.attn_backend.init_forward_metadata(self.static_batch)
        self.metadata = mr.attn_backend.forward_metadata
        self.graph = None
        if self.use_graph:
            with torch.inference_mode():
                self.new_lens.zero_()   # a step without a node: touches no request's state, page or cache row
                self._step()
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, pool=mr.graph_runner.pool if mr.graph_runner is not None else None):
                    self._step()
                self.graph = graph

    def _step(self) -> None:
        mr = self.mr
        ops.prepare_extend(self.req_pool_indices, self.prefix_lens, self.new_lens, self.alloc_lens, self.free_pages, self.free_range,
                           mr.req_to_token_pool.req_to_token, self.positions, self.out_cache_loc, self.cu_seqlens_q, self.seq_lens, self.status,
                           mr.page_size, parents=self.parents, tree_mask=self.tree_mask,
                           req_to_page=mr.req_to_token_pool.req_to_page if mr.page_size > 1 else None)
        mr.attn_backend.forward_metadata = self.metadata
        logits = mr.model(self.input_ids, self.positions, self.static_batch)
        target = ops.argmax(logits)
        if self.logprobs is not None:
            self._scores = ops.token_logprobs(logits, target, self.logprobs)
        ops.accept_tree(self.input_ids, target, self.parents, self.cu_seqlens_q, self.prefix_lens, self.out_cache_loc, self.layers, self.accept_lens,
                        self.accept_rows, self.accept_tokens, self.next_tokens, self.prefix_lens)

    # ------------------------------------------------------------------ a step
    @torch.inference_mode()
    def step(self, drafts: Sequence[Tuple[Sequence[int], Sequence[int]]]) -> List[List[int]]:
        """``drafts[b] = (tokens, parents)`` of request b's drafted nodes 1, 2, ...: node i drafts tokens[i - 1] behind node parents[i - 1] < i (0 =
        the request's last token).  Empty lists decode one token.  Returns the accepted tokens per request, appended to the requests too."""
        if len(drafts) != self.bs:
            raise ValueError(f"{len(drafts)} drafts for {self.bs} requests")
        self._take_lengths()
        ids, parents, lens = [], [], []
        for r, (tokens, par) in zip(self.batch.reqs, drafts):
            if len(tokens) != len(par) or len(tokens) >= self.max_nodes:
                raise ValueError(f"a draft has {len(tokens)} tokens and {len(par)} parents; at most {self.max_nodes - 1} nodes were announced")
            if any(not 0 <= p <= i for i, p in enumerate(par)):
                raise ValueError("a draft's parent must be an earlier node")
            if any(not 0 <= t < self.vocab for t in tokens):
                raise ValueError(f"a drafted token is outside the vocabulary of {self.vocab}")
            ids += [r.last_token_id, *tokens]
            parents += [-1, *par]
            lens.append(1 + len(tokens))
        if int(self.seq_lens_cpu.max()) + self.max_nodes > self.bound < self.mr.req_to_token_pool.req_to_token.shape[1]:
            self._prepare()
        if self._host_pages_changed():
            self._upload_free_list()  # only between a sync_host() and the next step
        n = len(ids)
        self.input_ids[:n].copy_(torch.tensor(ids, dtype=torch.int32))
        self.parents[:n].copy_(torch.tensor(parents, dtype=torch.int32))
        self.new_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        if self.graph is not None:
            self.graph.replay()
        else:
            self._step()
        status = int(self.status.item())
        if status:
            self.status.zero_()
            raise RuntimeError(f"tree step refused: {_REFUSED.get(status, status)}")
        self.pending += 1
        kept, tokens = self.accept_lens.tolist(), self.accept_tokens.tolist()
        out = [t[:k] for t, k in zip(tokens, kept)]
        if self._scores is not None:
            given, entropy, top_ids, top = (t.cpu() for t in self._scores)
            self.last_logprobs = [[(float(given[i]), float(entropy[i]), top_ids[i].tolist(), top[i].tolist()) for i in rows[:k]]
                                  for rows, k in zip(self.accept_rows.tolist(), kept)]
        self.seq_lens_cpu = self.seq_lens_cpu + torch.tensor(kept, dtype=self.seq_lens_cpu.dtype)
        for r, new in zip(self.batch.reqs, out):
            r.token_ids.extend(new)
        return out

    def sync_host(self) -> None:
        """Host state in line with the device: lengths, last slots, and the page allocator without the pages the contexts fill, those that
        rejected drafts had taken given back.  Decoding can go on by any other means afterwards, or here."""
        mr, b, ps = self.mr, self.batch, self.mr.page_size
        self._take_lengths()
        if self._host_pages_changed():
            self._upload_free_list()
        mr.page_allocator.alloc(int(self.free_range[0].item()))  # the same pages, in the same order, leave the host's free list
        table = mr.req_to_token_pool.req_to_token
        spare = []
        for i, r in enumerate(b.reqs):
            length, alloc = int(self.seq_lens_cpu[i]), int(self.alloc_lens[i])
            first = -(-length // ps) * ps
            if alloc > first:
                spare.append(table[r.req_pool_idx, first: alloc: ps].cpu() // ps)
            r.last_slot = int(table[r.req_pool_idx, length - 1])
        if spare:
            mr.page_allocator.free(torch.cat(spare))
        self.alloc_lens.copy_(self.prefix_lens)
        self._upload_free_list()
        b.seq_lens_cpu, self.synced_lens = self.seq_lens_cpu.clone(), self.seq_lens_cpu.clone()
        b.seq_lens = self.prefix_lens.clone()
        b.forward_mode = ForwardMode.DECODE
