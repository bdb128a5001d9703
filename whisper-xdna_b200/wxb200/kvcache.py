"""A paged key-value cache for a text decoder on the encoder's features: the
tensors that ops.kv_fork, kv_append, kv_compact and paged_attention work on, kept
together. Nothing here waits for the GPU.

A step of a decoder with beams:

    cache.step(parents, grow)          # beams reordered, ended, started; pages found
    for layer in range(cache.n_layers):
        cache.append(layer, k, v)      # this step's tokens
        o = cache.attend(layer, q)
"""
import torch

from . import ops


class PagedKVCache:
    """n_layers pools of n_pages pages of page_size tokens, for n_seqs sequences of
    up to max_len tokens (rounded up to whole pages). Tensors, all on `device`, by
    default the current one; calls are made with that device current:

    k, v: (n_layers, n_pages, page_size, n_heads, head_dim), uninitialised
    table: (n_seqs, width) int32 page table, -1 past a sequence's last page
    lens: (n_seqs,) int32 tokens, the last step's included
    refs: (n_pages,) int32 table entries that name a page, 0: free
    grown: (n_seqs,) int32 tokens that the last step granted
    status: int32 (pages left free, pages short) of the last step
    """

    def __init__(self, n_layers, n_pages, page_size, n_heads, head_dim, n_seqs, max_len,
                 dtype=torch.bfloat16, device=None):
        if min(n_layers, n_pages, page_size, n_heads, head_dim, n_seqs, max_len) < 1:
            raise ValueError("PagedKVCache: every size must be at least 1")
        device = torch.device("cuda" if device is None else device)
        if device.type != "cuda":
            raise ValueError(f"PagedKVCache: device must be a CUDA device, got {device}")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.n_layers, self.page_size, self.max_len = n_layers, page_size, max_len
        shape = (n_layers, n_pages, page_size, n_heads, head_dim)
        self.k = torch.empty(shape, dtype=dtype, device=device)
        self.v = torch.empty(shape, dtype=dtype, device=device)
        width = -(-max_len // page_size)
        i32 = dict(dtype=torch.int32, device=device)
        self.table = torch.full((n_seqs, width), -1, **i32)
        self.lens = torch.zeros(n_seqs, **i32)
        self.refs = torch.zeros(n_pages, **i32)
        self.grown = torch.zeros(n_seqs, **i32)
        self.status = torch.tensor([n_pages, 0], **i32)

    def step(self, parents=None, grow=None):
        """Sequence i goes on as parents[i] was (-1: it starts empty; None: as
        itself) with grow[i] more tokens (None: none): see ops.kv_fork. The table,
        lens, refs, grown and status are new tensors: a step captured in a CUDA graph
        to be replayed ends by copying the first three into those it began with."""
        self.table, self.lens, self.refs, self.grown, self.status = ops.kv_fork(
            self.k, self.v, self.table, self.lens, self.refs, parents=parents, grow=grow)

    def append(self, layer, k, v):
        """The tokens that the last step granted, all in one call: k, v (n_seqs, tokens,
        heads, head_dim), of which row t < grown[i] is used, or (n_seqs, heads,
        head_dim) after a step of one token at most. Fewer rows than grown[i] are
        written from the first granted position on, and reported by
        _lib.device_error as WX_DEVERR_PAGE: the others hold no token yet."""
        ops.kv_append(k, v, self.k[layer], self.v[layer], self.table, self.lens,
                      counts=self.grown)

    def attend(self, layer, q, **kw):
        """ops.paged_attention of one query token a sequence over a layer."""
        return ops.paged_attention(q, self.k[layer], self.v[layer], self.table, self.lens, **kw)

    def compact(self):
        """Moves the pages in use to the front of the pools."""
        self.table, self.refs, _ = ops.kv_compact(self.k, self.v, self.table, self.refs)
