"""Paged key/value cache: sequences share pages, and forking one costs a partly filled page at most.

A pool of pages [pages, blocks, 2, heads, page, dim] holds the keys (0) and values (1) of every full-attention block;
a page is 16, 32 or 64 consecutive tokens of a sequence in all blocks. Beside it, int32 on the same device: ``table``
[rows, width] lists each row's pages in order (-1 behind the last), ``lengths`` [rows] its tokens, ``refs`` [pages] how
many table entries hold a page (0: free). Nothing here reads them back to the host, so whole decode steps can be
captured as CUDA graphs.

The functions work on these tensors; ``PagedCache`` keeps them for a model. CUDA tensors run the kernels of
``csrc/paged``, CPU tensors ``ops.reference``. On CUDA the pool is bf16, heads have 64, 128 or 256 components, and
there are at most 1024 rows. An entry outside the pool is a page that is not there: what would be stored in it is
dropped, and attention does not see its tokens. None of them records gradients.
"""
import torch

from .ops import f32, native, reference

PAGES = (16, 32, 64)
DIMS = (64, 128, 256)


def _ints(name, part, shape, device):
    if part.dtype != torch.int32 or not part.is_contiguous():
        raise TypeError(f"{name} must be contiguous int32")
    if part.shape != shape:
        raise ValueError(f"{name} {tuple(part.shape)} does not match {tuple(shape)}")
    if part.device != device:
        raise ValueError(f"{name} is on {part.device}, the pool on {device}")


def _check(pool, table, lengths=None, refs=None, block=None):
    """What all functions ask of a cache's tensors (the CUDA calls check theirs in the extension, which is faster)."""
    shape, held, device = pool.shape, table.shape, pool.device
    if len(shape) != 6 or shape[2] != 2 or 0 in shape:
        raise ValueError(f"expected a pool [pages, blocks, 2, heads, page, dim], got {tuple(shape)}")
    if shape[4] not in PAGES:
        raise ValueError(f"a page holds {PAGES} tokens, got {shape[4]}")
    if not pool.is_contiguous():
        raise ValueError("the pool must be contiguous")
    if len(held) != 2 or 0 in held:
        raise ValueError(f"expected a table [rows, width], got {tuple(held)}")
    _ints("table", table, held, device)
    if lengths is not None:
        _ints("lengths", lengths, held[:1], device)
    if refs is not None:
        _ints("refs", refs, shape[:1], device)
    if block is not None and not 0 <= block < shape[1]:
        raise IndexError(f"block {block} of {shape[1]}")
    if pool.is_cuda:
        if pool.dtype != torch.bfloat16 or shape[5] not in DIMS:
            raise TypeError(f"the CUDA paged cache takes bf16 and head sizes {DIMS}, got {pool.dtype} and {shape[5]}")
        if held[0] > 1024:
            raise ValueError(f"the CUDA paged cache has at most 1024 rows, got {held[0]}")


def _check_rows(name, part, pool, table, shape):
    if part.shape != shape:
        raise ValueError(f"{name} {tuple(part.shape)} does not match {tuple(shape)}")
    if part.device != pool.device:
        raise ValueError(f"{name} is on {part.device}, the pool on {pool.device}")


def _check_out(given, to):
    """What is written may be the argument of its place, or lie apart from all of them and from the rest."""
    def apart(x, y):
        a, b = x.data_ptr(), y.data_ptr()
        return a >= b + y.nbytes or b >= a + x.nbytes

    for i, out in enumerate(to):
        if not all(apart(part, out) or i == j and part.data_ptr() == out.data_ptr() for j, part in enumerate(given)) or \
                not all(apart(other, out) for other in to[:i]):
            raise ValueError("out must be the arguments themselves or apart from them")


def check_parents(parents, rows, device):
    """[groups, beams] indices of each slot's parent within its group, ``rows`` slots in all."""
    if parents.dim() != 2 or parents.numel() != rows:
        raise ValueError(f"expected parents [groups, beams] of {rows} rows, got {tuple(parents.shape)}")
    if parents.dtype != torch.int64 or parents.device != device:
        raise TypeError(f"parents must be int64 on {device}")


def advance_pages(pool, table, lengths, refs, tokens=1, parents=None, live=None, out=None):
    """(table, lengths, refs, status) after every row took over its parent's history and got room for ``tokens`` more.

    ``parents`` [groups, beams] int64 (as ``beams.beam_select`` returns them; rows = groups * beams): a row continues
    the sequence of that slot of its group, whose pages it shares from then on. ``live`` (bool, one per row): the
    others give up their pages and have length 0. A new token goes behind the row's last one; where that page is
    partly filled and somebody else holds it too, its tokens are first copied into a page of the row's own (the last
    of the rows that share it keeps it). Pages are taken in order of rows, the lowest free one first. Of the pool
    only those copies are written.

    status [1] int32 has bit 1 if the pool ran out (the entry is -1), 2 if a row would outgrow its table (it keeps its
    length), 4 if a parent lies outside its group (the row keeps its own history). ``out``: (table, lengths, refs,
    status) to write to, which may be the arguments themselves; its status keeps the bits that it has."""
    if pool.is_cuda:
        return tuple(native().advance_pages(pool, table, lengths, refs, tokens, parents, live, out))
    _check(pool, table, lengths, refs)
    rows = table.shape[0]
    if not 0 <= tokens <= 1 << 30:
        raise ValueError(f"tokens must lie in 0..2^30, got {tokens}")
    if parents is not None:
        check_parents(parents, rows, pool.device)
    if live is not None:
        if live.dtype != torch.bool or live.numel() != rows or live.device != pool.device:
            raise ValueError(f"live must be {rows} bools on {pool.device}")
    if out is not None:
        _check(pool, out[0], out[1], out[2])
        if out[0].shape != table.shape or out[3].shape != (1,) or out[3].dtype != torch.int32 or \
                out[3].device != pool.device:
            raise ValueError("out must be (table, lengths, refs, status) like the arguments")
        _check_out((table, lengths, refs), out)
    result = reference.advance_pages(pool, table, lengths, refs, tokens, parents, live)
    if out is None:
        return result
    for to, part in zip(out[:3], result):
        to.copy_(part)
    out[3].bitwise_or_(result[3])
    return out


def compact_pages(pool, table, refs, out=None):
    """(table, refs, used): the pages in use moved to the front of the pool, whose first ``used`` [1] pages they are
    then. The lowest page behind them goes to the lowest free page among them, and so on; pages that lie there
    already stay. Pages that are held outside the table too move like the others. ``out``: (table, refs) to write to,
    which may be the arguments themselves."""
    if pool.is_cuda:
        return tuple(native().compact_pages(pool, table, refs, out))
    _check(pool, table, refs=refs)
    if out is not None:
        _check(pool, out[0], refs=out[1])
        if out[0].shape != table.shape:
            raise ValueError("out must be (table, refs) like the arguments")
        _check_out((table, refs), out)
    result = reference.compact_pages(pool, table, refs)
    if out is None:
        return result
    out[0].copy_(result[0])
    out[1].copy_(result[1])
    return out[0], out[1], result[2]


def store_pages(pool, block, table, lengths, keys, values):
    """Writes ``keys``, ``values`` [N, T, heads, dim] as the last T tokens of rows 0, R / N, 2 R / N, ... (the first of
    each group of beams); tokens before a row's first are dropped. For prompts, whose keys are rotated already."""
    if pool.is_cuda:
        return native().store_pages(pool, block, table, lengths, keys, values)
    _check(pool, table, lengths, block=block)
    if keys.dim() != 4 or keys.shape[0] < 1 or table.shape[0] % keys.shape[0]:
        raise ValueError(f"expected keys [rows / beams, tokens, heads, dim], got {tuple(keys.shape)}")
    shape = keys.shape[:2] + (pool.shape[3], pool.shape[5])
    _check_rows("keys", keys, pool, table, shape)
    _check_rows("values", values, pool, table, shape)
    reference.store_pages(pool, block, table, lengths, keys, values)


def append_heads(x, pool, block, table, lengths, q_weight, k_weight, inv_freq, heads, eps):
    """Queries [R, heads, dim] of each row's newest token, whose key and value go into the row's pages, in one pass.

    ``x`` [R, (2 heads + 2 pool heads) * dim] is the block's input projection: per query head [query | gate], then the
    keys, then the values. Queries and keys are normalised per head (times 1 + weight) and their first
    2 * len(inv_freq) components rotated to position lengths - 1, whose angle is formed in 64 bits. A row of length 0
    stores nothing."""
    if pool.is_cuda:
        return native().append_heads(x, pool, block, table, lengths, f32(q_weight), f32(k_weight), f32(inv_freq), heads,
                                     eps)
    _check(pool, table, lengths, block=block)
    D = pool.shape[5]
    if heads < 1 or heads % pool.shape[3]:
        raise ValueError(f"{heads} query heads for {pool.shape[3]} key heads")
    _check_rows("x", x, pool, table, (table.shape[0], (2 * heads + 2 * pool.shape[3]) * D))
    if q_weight.shape != (D,) or k_weight.shape != (D,) or inv_freq.dim() != 1 or 2 * len(inv_freq) > D:
        raise ValueError(f"expected weights of {D} and at most {D // 2} frequencies")
    if any(part.device != pool.device for part in (q_weight, k_weight, inv_freq)):
        raise ValueError(f"weights and frequencies must be on {pool.device}")
    return reference.append_heads(x, pool, block, table, lengths, q_weight, k_weight, inv_freq, heads, eps)


def paged_attention(q, pool, block, table, lengths, gate=None, group=1):
    """Attention [R, Hq, dim] of one token per row over the ``lengths`` tokens of its pages in one block, scaled by
    dim^-0.5; query head h reads key head h // (Hq / heads). ``gate`` [R, Hq, dim]: the result is multiplied by its
    sigmoid. A row without tokens has zeros. ``group``: that many consecutive rows are beams of one prompt; a page
    that several of them hold is read once (a matter of speed, and of the order in which sums are formed)."""
    if pool.is_cuda:
        return native().paged_attention(q, pool, block, table, lengths, gate, group)
    _check(pool, table, lengths, block=block)
    R, H, D = table.shape[0], pool.shape[3], pool.shape[5]
    if q.dim() != 3 or q.shape[1] < 1 or q.shape[1] % H or q.shape[1] > 64 * H:
        raise ValueError(f"expected q [rows, heads, dim] with 1 to 64 query heads per key head, got {tuple(q.shape)}")
    _check_rows("q", q, pool, table, (R, q.shape[1], D))
    if gate is not None:
        _check_rows("gate", gate, pool, table, q.shape)
    if group < 1 or R % group:
        raise ValueError(f"{R} rows are no groups of {group}")
    return reference.paged_attention(q, pool, block, table, lengths, gate)


class PagedCache:
    """The paged cache of a model's full-attention blocks: ``rows`` sequences of up to ``tokens`` tokens.

    ``pages``: the size of the pool. It is never overrun silently: ``check`` raises where a step did not find its
    pages."""

    def __init__(self, blocks, heads, dim, rows, tokens, pages, page=64, device="cpu", dtype=torch.bfloat16):
        if min(blocks, heads, dim, rows, tokens, pages) < 1:
            raise ValueError("a paged cache needs at least one block, head, component, row, token and page")
        self.page = page
        # zeros: attention reads whole tiles of a page
        self.pool = torch.zeros(pages, blocks, 2, heads, page, dim, device=device, dtype=dtype)
        self.table = torch.full((rows, -(-tokens // page)), -1, device=device, dtype=torch.int32)
        self.lengths = torch.zeros(rows, device=device, dtype=torch.int32)
        self.refs = torch.zeros(pages, device=device, dtype=torch.int32)
        self.status = torch.zeros(1, device=device, dtype=torch.int32)
        _check(self.pool, self.table, self.lengths, self.refs)

    def advance_(self, tokens=1, parents=None, live=None):
        """``advance_pages`` in place."""
        advance_pages(self.pool, self.table, self.lengths, self.refs, tokens, parents, live,
                      out=(self.table, self.lengths, self.refs, self.status))

    def free_(self, rows):
        """The rows of the bool mask ``rows`` give up their pages."""
        self.advance_(0, live=~rows)

    def compact_(self):
        """``compact_pages`` in place; returns the number of pages in use (waits for the device)."""
        return int(compact_pages(self.pool, self.table, self.refs, out=(self.table, self.refs))[2])

    def check(self):
        """Raises if a step since the last call went wrong (waits for the device)."""
        status = int(self.status)
        self.status.zero_()
        if status:
            what = ("the pool ran out of pages", "a row outgrew its table", "a parent lies outside its group")
            raise RuntimeError("paged cache: " + ", ".join(text for bit, text in enumerate(what) if status >> bit & 1))

    def store_(self, block, keys, values):
        store_pages(self.pool, block, self.table, self.lengths, keys, values)

    def append_(self, block, x, q_weight, k_weight, inv_freq, heads, eps):
        return append_heads(x, self.pool, block, self.table, self.lengths, q_weight, k_weight, inv_freq, heads, eps)

    def attend(self, block, q, gate=None, group=1):
        return paged_attention(q, self.pool, block, self.table, self.lengths, gate, group)

    def state_dict(self):
        """The pages in use (moved to the pool's front first), and who holds them."""
        used = self.compact_()
        return {"pages": self.pool[:used].clone(), "table": self.table.clone(), "lengths": self.lengths.clone(),
                "refs": self.refs[:used].clone()}

    def load_state_dict(self, state):
        used = state["pages"].shape[0]
        if state["table"].shape != self.table.shape or state["pages"].shape[1:] != self.pool.shape[1:] or \
                used > self.pool.shape[0]:
            raise ValueError("the saved pages do not fit this cache")
        self.pool[:used].copy_(state["pages"])
        self.refs.zero_()
        self.refs[:used].copy_(state["refs"])
        self.table.copy_(state["table"])
        self.lengths.copy_(state["lengths"])
        self.status.zero_()
