"""Token sequences: what an until-done loop over them does around its model.

A batch of sequences that each run until their own end is a batch of samples: the
``terminated`` mask and the compaction are the loop's own. Around the model's layers such
a loop, on the device and with nothing read back, needs

* the blocks of a paged cache that grown sequences take (:class:`BlockTables`, fed with
  the free list that ``compact`` makes of the used blocks' mask),
* the slots, positions and owners of the pass's new tokens (:class:`SlotMap`),
* the embedding rows of those tokens (:class:`Embedding`), and in training
* the gradient of the table (:class:`EmbeddingGrad`), whose sums, like the canonical
  reduction, have one order whatever the launch.

As with ``Compactor`` and ``Reducer`` a class prepares a call -- it checks the tensors,
holds them and allocates outputs and workspace once -- and calling it only enqueues
(and can be captured in a CUDA graph); the function of the same name prepares and calls.
Calls of one prepared object share its outputs and workspace: those that may overlap on
the GPU must be ordered by the caller, two graphs captured from it included, and so must a
call on another stream behind the preparation; one thread calls it at a time; a graph does
not keep the object, its owner does. No operator here records an autograd graph or carries
a tangent: tensors that ask for either are refused.
"""

from __future__ import annotations

import contextlib
import ctypes
import math

from . import _abi
from ._api import _ptr, _t

_TYPES = None


def _type(dtype, what, kinds):
    """The type code of a torch dtype, one of ``kinds`` ("element" or "index")."""
    torch = _t()
    global _TYPES
    if _TYPES is None:
        _TYPES = {"element": {torch.float32: _abi.TYPE_F32, torch.bfloat16: _abi.TYPE_BF16,
                              torch.float16: _abi.TYPE_F16},
                  "index": {torch.int32: _abi.TYPE_I32, torch.int64: _abi.TYPE_I64}}
    if dtype not in _TYPES[kinds]:
        raise TypeError(f"{what} must be {' or '.join(str(k).removeprefix('torch.') for k in _TYPES[kinds])}, "
                        f"not {dtype}")
    return _TYPES[kinds][dtype]


def _cuda(x, what, device=None):
    """``x``, a CUDA tensor (on ``device``)."""
    torch = _t()
    if not isinstance(x, torch.Tensor) or x.layout != torch.strided or not x.is_cuda:
        raise ValueError(f"{what} must be a CUDA tensor")
    if device is not None and x.device != device:
        raise ValueError(f"{what} is on {x.device}, not on {device}")
    _plain(x, what)
    return x


def _plain(x, what):
    """``x``'s memory holds its values (the imaginary part of a conjugate's holds their negatives)."""
    if x.is_neg():
        raise ValueError(f"{what} is a view that negates its memory: resolve it first (resolve_neg)")


def _whole(value, what):
    """``value`` as a whole number, one that the descs' 64 bits hold."""
    n = int(value)
    if n != value or not -2**63 <= n < 2**63:
        raise ValueError(f"{what} must be a whole number of at most 64 bits, not {value}")
    return n


def _no_grad(what, *tensors):
    torch = _t()
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError(f"{what} records no autograd graph: call it under torch.no_grad() or on detached tensors "
                         "(embedding_grad is the gradient of embedding)")
    if any(t is not None and torch.autograd.forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise ValueError(f"{what} carries no tangent: call it on the primal (forward_ad.unpack_dual), and embedding on "
                         "the tangent, which it is linear in")


def _extent(x):
    """The bytes from the first to the last element of ``x``."""
    if x.numel() == 0:
        return 0, 0
    last = sum((n - 1) * s for n, s in zip(x.shape, x.stride()))
    return x.data_ptr(), x.data_ptr() + (last + 1) * x.element_size()


def _beside(x, y):
    """Whether ``x`` and ``y`` lie in columns of one plane that do not meet: apart within every row of it."""
    pitch, runs = 0, []
    for t in (x, y):
        inner = t.dim() - 1 if t.dim() and t.stride(-1) == 1 else t.dim()  # the axes before a contiguous last one
        runs.append((t.shape[-1] if inner < t.dim() else 1) * t.element_size())
        for n, s in zip(t.shape[:inner], t.stride()):
            if n > 1:
                pitch = math.gcd(pitch, s * t.element_size())
    if pitch == 0:
        return False
    ahead = (y.data_ptr() - x.data_ptr()) % pitch
    return runs[0] <= ahead and ahead + runs[1] <= pitch


def _apart(out, what, *inputs):
    """``out`` shares no memory with the inputs."""
    lo, hi = _extent(out)
    for x in inputs:
        if x is not None:
            a, b = _extent(x)
            if lo < b and a < hi and not _beside(out, x):
                raise ValueError(f"{what} overlaps an input")


def _raw_stream(device):
    """The handle of ``device``'s current stream."""
    torch = _t()
    global _current
    if _current is None:  # the handle alone, where this torch offers it: a call a step makes every time
        _current = getattr(torch._C, "_cuda_getCurrentRawStream",
                           lambda index: torch.cuda.current_stream(index).cuda_stream)
    return _current(device.index)


_current = None


def _capturing(handle):
    flag = ctypes.c_int32()
    _abi.check(_abi.lib().eagle_backend_stream_is_capturing(handle, ctypes.byref(flag)))
    return bool(flag.value)


class _Call:
    """A prepared call: ``_desc`` and the C entry, enqueued on the tensors' device."""

    def _prepare(self, entry, desc, device, *tensors):
        self.device = device
        self._entry = getattr(_abi.lib(), entry)
        self._desc = desc
        self._ref = ctypes.byref(desc)
        self._tensors = [t for t in tensors if t is not None]  # what a call reads and writes
        self._home = _raw_stream(device)
        self._known = set()  # streams that the allocator knows to use them

    def _enqueue(self, stream):
        if stream is None:
            handle = _raw_stream(self.device)
        else:
            if stream.device != self.device:
                raise ValueError(f"the stream is on {stream.device}, the tensors on {self.device}")
            handle = stream.cuda_stream
        if (stream is not None or handle != self._home) and handle not in self._known and not _capturing(handle):
            # the allocator may hand the tensors' memory out again once they are dropped, the caller's too: not
            # before this stream is past the call (a capture runs nothing: what its graph uses, the graph's owner
            # keeps). Once a stream is enough: it is asked for how far it is when they are dropped
            s = stream if stream is not None else _t().cuda.current_stream(self.device)
            for t in self._tensors:
                t.record_stream(s)
            self._known.add(handle)
        self._desc.stream = handle
        status = self._entry(self._ref)
        if status:
            _abi.check(status)


def _on(stream):
    """Allocations on ``stream``, where the call runs."""
    return _t().cuda.stream(stream) if stream is not None else contextlib.nullcontext()


def _query(entry, desc, device):
    """The workspace that the call described by ``desc`` asks for."""
    torch = _t()
    _abi.check(getattr(_abi.lib(), entry)(ctypes.byref(desc)))
    work = torch.empty(max(int(desc.scratch_bytes), 256), dtype=torch.uint8, device=device)
    desc.scratch = _ptr(work)
    return work


# ------------------------------------------------------------------------- embedding

def _axes(tokens, values):
    """The tokens' axes as (batch, seq): sizes, and strides of the tokens and of their vectors. Neighbouring axes
    are joined where one stride serves both, in both tensors."""
    if tokens.numel() == 0:
        return [0, 1], [0, 0], [0, 0]
    joined = []
    for n, s, v in zip(tokens.shape, tokens.stride(), values.stride()):
        if n == 1:
            continue
        if joined and joined[-1][1:] == (n * s, n * v):
            joined[-1] = (joined[-1][0] * n, s, v)
        else:
            joined.append((n, s, v))
    if len(joined) > 2:
        raise ValueError(f"the {tokens.dim()} axes of the tokens must join into two, for them and their vectors alike "
                         "(reshape them)")
    return tuple(zip(*([(1, 0, 0)] * (2 - len(joined)) + joined)))


def _embedding_desc(table, values, tokens, rows, scale, first, device):
    torch = _t()
    dim = values.shape[-1]
    shape, token_strides, value_strides = _axes(tokens, values)
    d = _abi.new(_abi.EmbeddingDesc, device=device.index, table_type=_type(table.dtype, "the table", "element"),
                 values_type=_type(values.dtype, "the tokens' vectors", "element"),
                 token_type=_type(tokens.dtype, "tokens", "index"), table=_ptr(table), tokens=_ptr(tokens),
                 values=_ptr(values), rows=rows, dim=dim, first=_whole(first, "first"), batch=shape[0], seq=shape[1],
                 table_stride=max(table.stride(0), dim), scale=float(scale))
    d.token_strides[:] = token_strides
    d.value_strides[:] = [*value_strides, values.stride(-1)]
    return d


def _check_out(out, shape, dtype, device, what):
    """``out``: ``shape`` vectors that lie apart, their values contiguous."""
    _cuda(out, what, device)
    if tuple(out.shape) != tuple(shape) or (dtype is not None and out.dtype != dtype):
        raise ValueError(f"{what} must be a tensor of shape {tuple(shape)}" + (f" and {dtype}" if dtype else ""))
    if out.numel() == 0:
        return out
    room = 1
    for size, stride in sorted(((n, s) for n, s in zip(out.shape, out.stride()) if n > 1), key=lambda ns: ns[1]):
        if stride < room:
            raise ValueError(f"the elements of {what} overlap")
        room = (size - 1) * stride + room
    if out.shape[-1] > 1 and out.stride(-1) != 1:
        raise ValueError(f"the vectors of {what} must be contiguous")
    return out


class Embedding(_Call):
    """A prepared lookup: ``out[..., :] = scale * table[tokens - first, :]``, the product in
    32 bits, rounded once to ``out``'s type.

    ``table`` is (rows, dim), float32, bfloat16 or float16, each row contiguous; the rows
    may lie apart (a slice of a wider or longer one). ``tokens`` are int32 or int64 of any
    shape; their axes must join into two, each of one stride (two axes or fewer always do).
    A token outside ``[first, first + rows)`` -- padding marked -1, a row
    that another rank's shard holds -- gives zeros. ``out`` (or its ``dtype``, by default the
    table's) may be any of the three types. Calls return ``out``, of shape
    ``(*tokens.shape, dim)``."""

    def __init__(self, table, tokens, *, scale: float = 1.0, first: int = 0, out=None, dtype=None):
        torch = _t()
        _cuda(table, "the table")
        device = table.device
        _cuda(tokens, "tokens", device)
        if table.dim() != 2 or (table.numel() > 0 and table.shape[1] > 1 and table.stride(1) != 1):
            raise ValueError("the table must be (rows, dim) with contiguous rows")
        if table.numel() > 0 and table.shape[0] > 1 and table.stride(0) < table.shape[1]:
            raise ValueError("the table's rows overlap")
        _no_grad("embedding", table, out)
        shape = (*tokens.shape, table.shape[1])
        _type(tokens.dtype, "tokens", "index")
        _type(dtype or table.dtype, "the table and dtype", "element")
        if out is None:
            out = torch.empty(shape, dtype=dtype or table.dtype, device=device)
        else:
            _check_out(out, shape, dtype, device, "out")
            _apart(out, "out", table, tokens)
        self.table, self.tokens, self.out = table, tokens, out
        d = _embedding_desc(table, out, tokens, table.shape[0], scale, first, device)
        self._prepare("eagle_backend_x_b200_embedding", d, device, table, tokens, out)

    def __call__(self, stream=None):
        self._enqueue(stream)
        return self.out


def embedding(table, tokens, *, scale: float = 1.0, first: int = 0, out=None, dtype=None, stream=None):
    """``scale * table[tokens - first]``, zeros for tokens the table has no row for (:class:`Embedding`)."""
    with _on(stream):
        return Embedding(table, tokens, scale=scale, first=first, out=out, dtype=dtype)(stream)


class EmbeddingGrad(_Call):
    """The prepared gradient of :class:`Embedding` with respect to its table:
    ``out[v, :] = scale *`` the sum of ``grad[..., :]`` over the tokens equal to
    ``first + v``, and zeros for a row without a token.

    ``grad`` is ``(*tokens.shape, dim)``, float32, bfloat16 or float16, with any strides, a
    broadcast's zeros included (of more than two leading axes: that join into two where the
    tokens' do). ``out`` is (rows, dim), contiguous rows, of ``dtype`` (by
    default ``grad``'s). Padding is left out where it is marked by an id that the table has no
    row for (-1); an id of one of its rows is summed, whatever it stands for. With
    ``accumulate`` the sums are added to ``out`` (required then):
    rows without a token stay as they are. Each row is summed in 32 bits in one order that
    the sizes alone fix and rounded once, so the bits do not depend on the launch. The
    workspace is about 16 bytes a token and a 32-bit row per 4 to 32 tokens.

    The waits for rows on their way are bounded. Should one run out, the rows of ``out`` that
    needed them hold NaN, and :meth:`check` says so."""

    def __init__(self, grad, tokens, rows: int, *, scale: float = 1.0, first: int = 0, out=None, dtype=None,
                 accumulate: bool = False):
        torch = _t()
        _cuda(grad, "grad")
        device = grad.device
        _cuda(tokens, "tokens", device)
        if grad.dim() != tokens.dim() + 1 or grad.shape[:-1] != tokens.shape:
            raise ValueError(f"grad must be of shape (*tokens.shape, dim), got {tuple(grad.shape)} for "
                             f"{tuple(tokens.shape)} tokens")
        _no_grad("embedding_grad", grad, out)
        _type(tokens.dtype, "tokens", "index")
        _type(grad.dtype, "grad", "element")
        rows = _whole(rows, "rows")
        if rows < 0:
            raise ValueError("rows must not be negative")
        shape = (rows, grad.shape[-1])
        if out is None:
            if accumulate:
                raise ValueError("accumulate adds to out: give it")
            _type(dtype or grad.dtype, "dtype", "element")
            out = torch.empty(shape, dtype=dtype or grad.dtype, device=device)
        else:
            _check_out(out, shape, dtype, device, "out")
            _apart(out, "out", grad, tokens)
        self.grad, self.tokens, self.out = grad, tokens, out
        d = _embedding_desc(out, grad, tokens, rows, scale, first, device)
        d.flags = _abi.EMBEDDING_ACCUMULATE if accumulate else 0
        self._work = _query("eagle_backend_x_b200_embedding_grad", d, device)
        self._prepare("eagle_backend_x_b200_embedding_grad", d, device, grad, tokens, out, self._work)

    def __call__(self, stream=None):
        self._enqueue(stream)
        return self.out

    def check(self, stream=None):
        """Wait for ``stream`` (by default the current one) and raise :class:`BackendError` if a wait of the last
        call, which it is past then, ran out."""
        if self.tokens.numel() == 0 or self.out.numel() == 0:
            return
        torch = _t()
        with torch.cuda.stream(stream if stream is not None else torch.cuda.current_stream(self.device)):
            lost = int(self._work[:4].view(torch.int32).item())
        if lost:
            raise _abi.BackendError(_abi.ERROR, "embedding_grad: a wait for rows ran out; the rows that needed them "
                                                "are NaN")


def embedding_grad(grad, tokens, rows: int, *, scale: float = 1.0, first: int = 0, out=None, dtype=None,
                   accumulate: bool = False, stream=None):
    """The gradient of :func:`embedding`'s table from that of its output (:class:`EmbeddingGrad`)."""
    with _on(stream):
        return EmbeddingGrad(grad, tokens, rows, scale=scale, first=first, out=out, dtype=dtype,
                             accumulate=accumulate)(stream)


# ------------------------------------------------------------------------- paged cache

def _vector(x, n, dtypes, device, what):
    """``x``: a contiguous vector of ``n`` (any number if None) of one of ``dtypes``."""
    _cuda(x, what, device)
    if x.dtype not in dtypes:
        raise TypeError(f"{what} must be {' or '.join(str(k).removeprefix('torch.') for k in dtypes)}, not {x.dtype}")
    if x.dim() != 1 or not x.is_contiguous() or (n is not None and x.numel() != n):
        raise ValueError(f"{what} must be a contiguous vector" + (f" of {n}" if n is not None else ""))
    return x


def _paged_desc(table, lengths, block, terminated, what):
    torch = _t()
    _cuda(table, "the table")
    device = table.device
    if table.dtype != torch.int32:
        raise TypeError(f"the table must be int32, not {table.dtype}")
    if table.dim() != 2 or (table.numel() > 0 and ((table.shape[1] > 1 and table.stride(1) != 1)
                                                   or (table.shape[0] > 1 and table.stride(0) < table.shape[1]))):
        raise ValueError("the table must be (requests, width), its rows contiguous and apart")
    requests, width = table.shape
    _vector(lengths, requests, (torch.int32, torch.int64), device, what)
    if terminated is not None:
        _vector(terminated, requests, (torch.bool, torch.uint8), device, "terminated")
    return _abi.new(_abi.PagedDesc, device=device.index, length_type=_type(lengths.dtype, what, "index"),
                    requests=requests, width=width, table_stride=max(table.stride(0), width), block=_whole(block, "block"),
                    table=_ptr(table), terminated=_ptr(terminated) if terminated is not None else 0)


class BlockTables(_Call):
    """The prepared growth of a paged cache's block tables.

    Row r of ``table`` (int32, (requests, width)) names the blocks, of ``block`` places
    each, that hold request r's tokens; ``held`` (int32) says how many it has.
    Calls give every live request the blocks that ``lengths`` (int32 or int64; the tokens
    it is to have room for) needs past those, in request order, off the front of ``pool``
    (int32), of which ``count`` (one int32, on the device) ids are valid:
    ``pool, count = compact(used)`` is the free list of a ``used`` mask, lowest ids first.
    A call writes the ids into ``table`` and sets their bytes in ``used`` (bool or uint8,
    if given). Requests set in ``terminated`` give their blocks back: their bytes in
    ``used`` are cleared. It returns ``(blocks, cells)``: the blocks each request has now
    (``held`` for the next call) and int32 ``[taken, short]``.

    A request is *short*, and keeps what it holds, when its row is too narrow or the pool,
    less what the requests before it asked for, too small. Entries of a row past what its
    request holds are left as they were, given back ones included: :class:`SlotMap` takes
    ``blocks`` to pass over them. ``held`` and ``pool`` are not
    written, so a call repeated on the same inputs gives the same result. Copy ``blocks`` to
    ``held`` before the free list is made again: a terminated request whose old count stays
    gives the same blocks back in every call, whoever has them by then, and an id that is in
    the pool and given back too is set and cleared in no order. No two requests share a block."""

    def __init__(self, lengths, held, table, pool, count, *, block: int, used=None, terminated=None):
        torch = _t()
        d = _paged_desc(table, lengths, block, terminated, "lengths")
        device, requests = table.device, table.shape[0]
        _vector(held, requests, (torch.int32,), device, "held")
        _vector(pool, None, (torch.int32,), device, "pool")
        _cuda(count, "count", device)
        if count.dtype not in (torch.int32, torch.uint32) or count.numel() != 1:
            raise ValueError("count must be one int32")
        if used is not None:
            _vector(used, None, (torch.bool, torch.uint8), device, "used")
        for out, what in ((table, "the table"), (used, "used")):
            if out is not None:
                _apart(out, what, lengths, held, pool, count, terminated)
        if used is not None:
            _apart(used, "used", table)
        self.lengths, self.held, self.table, self.pool, self.count = lengths, held, table, pool, count
        self.used, self.terminated = used, terminated
        self.blocks = torch.empty(requests, dtype=torch.int32, device=device)
        self.cells = torch.empty(2, dtype=torch.int32, device=device)
        d.lengths, d.held, d.pool, d.count, d.pool_size = (_ptr(lengths), _ptr(held), _ptr(pool), _ptr(count),
                                                           pool.numel())
        if used is not None:
            d.used, d.used_size = _ptr(used), used.numel()
        d.blocks, d.cells = _ptr(self.blocks), _ptr(self.cells)
        self._work = _query("eagle_backend_x_b200_block_tables", d, device)
        self._prepare("eagle_backend_x_b200_block_tables", d, device, lengths, held, table, pool, count, used,
                      terminated, self.blocks, self.cells, self._work)

    def __call__(self, stream=None):
        self._enqueue(stream)
        return self.blocks, self.cells


def block_tables(lengths, held, table, pool, count, *, block: int, used=None, terminated=None, stream=None):
    """Grow ``table`` to ``lengths`` from the free ``pool``: ``(blocks, cells)`` (:class:`BlockTables`)."""
    with _on(stream):
        return BlockTables(lengths, held, table, pool, count, block=block, used=used, terminated=terminated)(stream)


class SlotMap(_Call):
    """The prepared slots of a pass's new tokens, packed in request order.

    Live request r adds ``fresh[r]`` tokens from position ``start[r]`` on (both int32, or
    both int64). Calls return ``(slots, positions, requests, offsets)``: for each
    packed token its slot ``table[r, position // block] * block + position % block``
    (``dtype`` int64 or int32), its position (``start``'s type) and its request (int32), and
    int32 ``offsets`` of requests + 1 entries, request r's tokens being
    ``offsets[r]:offsets[r + 1]``. A token whose position lies past the table's width, whose
    block is not there (a negative entry) or whose slot does not fit ``dtype`` has slot -1;
    with ``held`` (int32: the blocks each request holds, ``BlockTables.blocks``) also one
    whose position lies past those. Give it wherever a row of the table serves one request
    after the other: without, a request left short takes what the one before left there.

    The first three have ``capacity`` entries whatever the number of tokens, so that a
    captured graph can serve any batch: entries past the last token have slot -1, position
    0 and request -1 (:class:`Embedding` gives zeros for a token marked -1); tokens past
    ``capacity`` are left out, which ``offsets`` shows."""

    def __init__(self, table, start, fresh, capacity: int, *, block: int, held=None, terminated=None, dtype=None):
        torch = _t()
        d = _paged_desc(table, start, block, terminated, "start")
        device, requests = table.device, table.shape[0]
        _vector(fresh, requests, (start.dtype,), device, "fresh")
        if held is not None:
            _vector(held, requests, (torch.int32,), device, "held")
            d.held, d.flags = _ptr(held), _abi.SLOT_MAP_HELD
        dtype = dtype or torch.int64
        d.slot_type = _type(dtype, "dtype", "index")
        capacity = _whole(capacity, "capacity")
        if capacity < 0:
            raise ValueError("capacity must not be negative")
        self.table, self.start, self.fresh, self.held, self.terminated = table, start, fresh, held, terminated
        d.capacity = capacity
        d.start, d.fresh = _ptr(start), _ptr(fresh)
        self._work = _query("eagle_backend_x_b200_slot_map", d, device)  # refuses before anything is allocated
        self.slots = torch.empty(capacity, dtype=dtype, device=device)
        self.positions = torch.empty(capacity, dtype=start.dtype, device=device)
        self.requests = torch.empty(capacity, dtype=torch.int32, device=device)
        self.offsets = torch.empty(requests + 1, dtype=torch.int32, device=device)
        d.slots, d.positions, d.token_requests, d.offsets = (_ptr(self.slots), _ptr(self.positions),
                                                             _ptr(self.requests), _ptr(self.offsets))
        self._prepare("eagle_backend_x_b200_slot_map", d, device, table, start, fresh, held, terminated, self.slots,
                      self.positions, self.requests, self.offsets, self._work)

    def __call__(self, stream=None):
        self._enqueue(stream)
        return self.slots, self.positions, self.requests, self.offsets


def slot_map(table, start, fresh, capacity: int, *, block: int, held=None, terminated=None, dtype=None, stream=None):
    """The packed new tokens' ``(slots, positions, requests, offsets)`` (:class:`SlotMap`)."""
    with _on(stream):
        return SlotMap(table, start, fresh, capacity, block=block, held=held, terminated=terminated,
                       dtype=dtype)(stream)
