"""Operators of a reader model that answers from retrieved passages, in the codes of the int4 corpora.

``Int4KVCache`` holds keys and values as symmetric 4-bit codes with one fp32 scale per vector (one token, one
head), the layout of a corpus packed as ``int4_per_token``.  Tokens are written as they are produced, read back,
moved, and attended to where they lie, under a window with first tokens that stay visible and for trees of drafted
tokens (``draft_ancestors``) too.  ``PageTable`` keeps which pages sequences own, ``Rotary`` turns queries and keys by
their positions, ``Int4Linear`` multiplies a few rows with 4-bit weights.  All take and return CUDA tensors, run on
torch's current stream without synchronising, allocate through torch only, and can be captured into a CUDA graph.

There is no backward pass: these are the operators of serving.  A query, keys to rotate or rows that require a gradient
are refused while gradients are enabled; codes, scales and a bias are constants, and keys and values are quantised
without one.
"""

from __future__ import annotations

import ctypes
from fractions import Fraction

torch = _lib = lib = check = _native = None


def _load():
    """Import torch, the CUDA library and the module between them, once, when the first object is made (the package
    imports without them)."""
    global torch, _lib, lib, check, _native
    if _native is None:
        import torch as torch_module
        from maxsim_b200 import _lib as lib_module

        try:
            from maxsim_b200 import _generation
        except ImportError as error:
            raise ImportError("maxsim_b200/_generation.so is missing or does not load: build it with "
                              "`python -m maxsim_b200.build`") from error
        torch, _lib, lib, check = torch_module, lib_module, lib_module.lib, lib_module.check
        _native = _generation


def _type_id(dtype, allowed="fp32, fp16 or bf16"):
    ids = {torch.float16: _lib.TYPE_F16, torch.bfloat16: _lib.TYPE_BF16}
    if "fp32" in allowed:
        ids[torch.float32] = _lib.TYPE_F32
    if dtype not in ids:
        raise ValueError(f"dtype must be {allowed}, got {dtype}")
    return ids[dtype]


def _on(tensor, name, device, dtype=None, ndim=None):
    if not hasattr(tensor, "data_ptr"):
        raise TypeError(f"{name} must be a torch tensor")
    if tensor.device != device:
        raise ValueError(f"{name} must be on {device}, got {tensor.device}")
    if dtype is not None and tensor.dtype != dtype:
        raise ValueError(f"{name} must have dtype {dtype}, got {tensor.dtype}")
    if ndim is not None and tensor.dim() != ndim:
        raise ValueError(f"{name} must have {ndim} dimensions, got {tensor.dim()}")
    return tensor


class Int4KVCache:
    """Keys and values of a model's layer as 4-bit codes, in pages.

    ``num_pages`` pages of ``page_size`` tokens (a power of two, 16 to 1024); ``head_dim`` 64, 128 or 256.  Slot
    ``s`` is token ``s % page_size`` of page ``s // page_size``; which pages a sequence owns, and in what order,
    is the caller's (``page_table``).  ``k_codes`` / ``v_codes`` are uint8 ``[pages, kv_heads, page_size,
    head_dim / 2]`` (even dimension in the low nibble), ``k_scales`` / ``v_scales`` fp32 ``[pages, kv_heads,
    page_size]``.  A vector takes ``head_dim / 2 + 4`` bytes.
    """

    def __init__(self, num_pages, page_size, num_kv_heads, head_dim, *, device="cuda"):
        _load()
        if min(int(num_pages), int(num_kv_heads)) < 1:
            raise ValueError("num_pages and num_kv_heads must be positive")
        shape = (int(num_pages), int(num_kv_heads), int(page_size))
        _check_cache_sizes(int(page_size), int(head_dim))
        codes = [torch.zeros(shape + (int(head_dim) // 2,), dtype=torch.uint8, device=device) for _ in range(2)]
        scales = [torch.ones(shape, dtype=torch.float32, device=device) for _ in range(2)]
        self._bind(codes[0], scales[0], codes[1], scales[1])

    @classmethod
    def from_tensors(cls, k_codes, k_scales, v_codes, v_scales):
        """A cache over arrays the caller owns (shapes above, contiguous).  Codes are those of `append`: a vector's largest
        is 7 or near it, a vector of zeros has scale 1 (or 0)."""
        self = cls.__new__(cls)
        self._bind(k_codes, k_scales, v_codes, v_scales)
        return self

    def _bind(self, k_codes, k_scales, v_codes, v_scales):
        _load()
        if not hasattr(k_codes, "data_ptr") or k_codes.dim() != 4:
            raise ValueError("k_codes must have shape [pages, kv_heads, page_size, head_dim / 2]")
        device = k_codes.device
        if device.type != "cuda":
            raise ValueError(f"the cache must be on a CUDA device, got {device}")
        for name, t, dtype, shape in (("k_codes", k_codes, torch.uint8, k_codes.shape),
                                      ("v_codes", v_codes, torch.uint8, k_codes.shape),
                                      ("k_scales", k_scales, torch.float32, k_codes.shape[:3]),
                                      ("v_scales", v_scales, torch.float32, k_codes.shape[:3])):
            _on(t, name, device, dtype)
            if t.shape != shape:
                raise ValueError(f"{name} must have shape {list(shape)}, got {list(t.shape)}")
            if not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous")
        pages, heads, size, half = k_codes.shape
        _check_cache_sizes(size, 2 * half)
        if pages < 1 or heads < 1:
            raise ValueError("num_pages and num_kv_heads must be positive")
        if any(t.data_ptr() % 16 for t in (k_codes, k_scales, v_codes, v_scales)):
            raise ValueError("cache arrays must be 16-byte aligned")
        self._arrays = (k_codes, k_scales, v_codes, v_scales)
        self.device = device
        self.num_pages, self.num_kv_heads, self.page_size, self.head_dim = pages, heads, size, 2 * half
        self._c = _lib.Kv4Cache(k_codes.data_ptr(), k_scales.data_ptr(), v_codes.data_ptr(), v_scales.data_ptr(), pages,
                                size, heads, 2 * half, device.index)
        self._address = ctypes.addressof(self._c)

    # Read-only: the kernels use the addresses of the arrays that the cache was made with.
    k_codes = property(lambda self: self._arrays[0])
    k_scales = property(lambda self: self._arrays[1])
    v_codes = property(lambda self: self._arrays[2])
    v_scales = property(lambda self: self._arrays[3])

    @property
    def resident_bytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self._arrays)

    def append(self, keys, values, slots) -> None:
        """Quantise ``keys`` and ``values`` ``[tokens, kv_heads, head_dim]`` (fp32, fp16 or bf16, any token and
        head strides) into int64 ``slots`` ``[tokens]``.

        Per vector: ``scale = max|x| * fl(1/7)`` (0 becomes 1), ``code = clip(rint(x / scale), -7, 7)``.  A vector with
        a value that is not finite stores scale NaN and codes 0.  A slot outside the cache (-1, say) is skipped; a
        slot must not be given twice in one call."""
        _native.append(self._address, keys, values, slots)

    def read(self, slots, *, dtype=None, out=None):
        """``(keys, values)`` of int64 ``slots`` as ``[tokens, kv_heads, head_dim]`` of ``dtype`` (bf16 by default):
        ``code * scale`` rounded once; zeros for a slot outside the cache.  ``out``: a pair of contiguous tensors
        on 16-byte boundaries."""
        return _native.read(self._address, slots, dtype, out)

    def slots(self, page_table, sequences, positions):
        """int64 slots of ``positions`` of ``sequences`` (tensors of one shape) under ``page_table``; -1, which `append`
        skips, where the table has no such sequence or position (a negative one is padding) or names no page."""
        sequences, positions = sequences.long(), positions.long()
        batch, width = page_table.shape
        if page_table.numel() == 0:
            return positions.new_full(positions.shape, -1)
        column = positions // self.page_size
        row_held, column_held = sequences.clamp(0, batch - 1), column.clamp(0, width - 1)
        known = (sequences == row_held) & (column == column_held)
        slot = (positions % self.page_size).add(page_table[row_held, column_held].long(), alpha=self.page_size)
        return slot.clamp(min=-1).where(known, -1)

    def move(self, source, target) -> None:
        """Copy the cached vectors of int64 slots ``source`` ``[tokens]`` to ``target`` ``[tokens]``, as if every source
        were read before any target is written: an accepted path of drafted tokens takes the places after the context's
        last token, a prefix is copied for another sequence.  A pair with either slot outside the cache (-1, say) is
        skipped; a target must not be given twice in one call."""
        _native.move(self._address, source, target)

    def attend(self, query, page_table, lengths, *, query_offsets=None, max_query_tokens=None, scale=None, causal=True,
               window=None, sinks=0, ancestors=None, return_lse=False, out=None):
        """Attention of ``query`` ``[rows, heads, head_dim]`` (fp16 or bf16) over cached tokens.

        ``lengths`` int32 ``[batch]`` counts each sequence's cached tokens, the rows' own among them; int32
        ``page_table`` ``[batch, max_pages]`` names their pages.  Sequence ``b`` owns rows ``query_offsets[b] ..
        query_offsets[b + 1]`` (int32 ``[batch + 1]``, at most ``max_query_tokens`` each), which are its last
        positions; without ``query_offsets`` each sequence has one row.  Rows before the first offset and past the last
        (padding) are zeros, rows past their sequence's ``max_query_tokens`` NaN; a given ``out`` keeps what it holds
        in both (and their log-sum-exp is -inf).  ``max_query_tokens`` defaults to all rows, and the kernel is chosen for
        as many in every sequence: give it where sequences share the rows.

        A row at position ``p`` sees tokens up to ``p`` (``causal``; otherwise all of its sequence), the last
        ``window`` of them where a window is given, and, ``sinks`` given beside it, the first ``sinks`` ones.

        ``ancestors`` int64 ``[rows, words]`` makes a sequence's rows the nodes of a tree of drafted tokens: a row sees
        those of its sequence's rows whose bit it has (bit ``k % 64`` of word ``k // 64``, from `draft_ancestors`; its own
        bit too), and all that is cached before them, or, with a window, the last ``window - n`` of it, ``n`` its bits, and
        the sinks.

        ``heads`` is a multiple of the cache's heads, consecutive
        query heads share one.  ``scale`` defaults to ``head_dim ** -0.5``.  A row that sees nothing is zero.
        Returns ``[rows, heads, head_dim]`` in the query's dtype, with ``return_lse`` also the fp32 natural
        log-sum-exp ``[rows, heads]`` (-inf where nothing is seen), with which results over parts of a context
        can be joined.  ``out`` may be the (contiguous) query itself, but not overlap it otherwise."""
        return _native.attend(self._address, query, page_table, lengths, query_offsets, max_query_tokens, scale, causal,
                              window, sinks, ancestors, return_lse, out)


def _check_cache_sizes(page_size, head_dim):
    if head_dim not in (64, 128, 256):
        raise ValueError(f"head_dim must be 64, 128 or 256, got {head_dim}")
    _check_page_size(page_size)


def draft_ancestors(parents, query_offsets, *, max_query_tokens=None):
    """``(ancestors, depths)`` of the nodes of drafted trees, one tree a sequence.

    ``parents`` int32 ``[rows]``: a node's parent as a row of its sequence, counted from the sequence's first and before
    the node; -1 (any other number) for a node that follows the context's last token.  Sequence ``b`` owns rows
    ``query_offsets[b] .. query_offsets[b + 1]`` (int32 ``[batch + 1]``, at most ``max_query_tokens`` each, which defaults
    to all rows and is at most 1024).  ``ancestors`` int64 ``[rows, ceil(max_query_tokens / 64)]``: the nodes on the path
    from the context to the row, itself among them, as `Int4KVCache.attend` takes them; ``depths`` int32 ``[rows]``: how
    many are above it, so that its position is its sequence's context length plus that.  Rows that no sequence owns, and
    those past their sequence's ``max_query_tokens``, get 0."""
    _load()
    return _native.draft_ancestors(parents, query_offsets, max_query_tokens)


class PageTable:
    """Which pages of a cache the sequences of a batch own, kept on the device.

    ``max_sequences`` sequences of up to ``max_pages`` pages of ``page_size`` tokens (a power of two, 16 to 1024) share
    ``num_pages`` pages.  ``page_table`` int32 ``[max_sequences, max_pages]`` (-1 where there is none) and ``lengths``
    int32 ``[max_sequences]`` are what `Int4KVCache.attend` takes; pages that no sequence owns lie on a stack,
    ``free_pages`` int32 ``[num_pages]`` of which the first ``free_count`` (int32 ``[1]``) are valid.  A page belongs to
    one sequence.  All four change in place, so calls on one table must not overlap on the GPU (one stream, or an order
    between streams)."""

    def __init__(self, num_pages, page_size, max_sequences, max_pages, *, device="cuda"):
        _load()
        if min(int(num_pages), int(max_sequences), int(max_pages)) < 1:
            raise ValueError("num_pages, max_sequences and max_pages must be positive")
        _check_page_size(int(page_size))
        if torch.device(device).type != "cuda":
            raise ValueError(f"the page table must be on a CUDA device, got {device}")
        self._bind(torch.full((int(max_sequences), int(max_pages)), -1, dtype=torch.int32, device=device),
                   torch.zeros(int(max_sequences), dtype=torch.int32, device=device),
                   torch.arange(int(num_pages) - 1, -1, -1, dtype=torch.int32, device=device),
                   torch.full((1,), int(num_pages), dtype=torch.int32, device=device), int(page_size))

    @classmethod
    def from_tensors(cls, page_table, lengths, free_pages, free_count, *, page_size):
        """A page table over arrays the caller owns (shapes above, contiguous)."""
        self = cls.__new__(cls)
        self._bind(page_table, lengths, free_pages, free_count, int(page_size))
        return self

    def _bind(self, page_table, lengths, free_pages, free_count, page_size):
        _load()
        if not hasattr(page_table, "data_ptr") or page_table.dim() != 2:
            raise ValueError("page_table must have shape [max_sequences, max_pages]")
        device = page_table.device
        if device.type != "cuda":
            raise ValueError(f"the page table must be on a CUDA device, got {device}")
        for name, t, ndim in (("page_table", page_table, 2), ("lengths", lengths, 1), ("free_pages", free_pages, 1),
                              ("free_count", free_count, 1)):
            _on(t, name, device, torch.int32, ndim)
            if not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous")
        sequences, columns = page_table.shape
        if lengths.shape[0] != sequences or free_count.shape[0] != 1:
            raise ValueError(f"lengths must have shape [{sequences}], free_count [1]")
        if min(sequences, columns, free_pages.shape[0]) < 1:
            raise ValueError("num_pages, max_sequences and max_pages must be positive")
        _check_page_size(page_size)
        if columns * page_size > 2**31 - 65536:
            raise ValueError("max_pages * page_size must be at most 2^31 - 65536")
        if max(sequences, free_pages.shape[0]) >= 2**31:
            raise ValueError("num_pages and max_sequences must be below 2^31")
        arrays = (page_table, lengths, free_pages, free_count)
        spans = sorted((t.data_ptr(), t.data_ptr() + 4 * t.numel()) for t in arrays)
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError("the page table's arrays must not overlap")
        self._arrays = arrays
        self.device = device
        self.num_pages, self.page_size = free_pages.shape[0], page_size
        self.max_sequences, self.max_pages = sequences, columns
        self._c = _lib.PageTableArrays(*(t.data_ptr() for t in arrays), self.num_pages, sequences, columns, page_size,
                                       device.index)
        self._address = ctypes.addressof(self._c)

    # Read-only: the kernels use the addresses of the arrays that the table was made with.
    page_table = property(lambda self: self._arrays[0])
    lengths = property(lambda self: self._arrays[1])
    free_pages = property(lambda self: self._arrays[2])
    free_count = property(lambda self: self._arrays[3])

    def extend(self, tokens, rows):
        """Give sequence ``b`` ``tokens[b]`` more tokens (int32 ``[max_sequences]``, 0 or less: none) and the pages that
        they need.  Returns ``(query_offsets, slots, positions)`` of the step's ``rows`` rows (a number that the host
        knows, the tokens' sum or more), which lie in the sequences' order: int32 ``[max_sequences + 1]``, int64
        ``[rows]`` (for `Int4KVCache.append`), int32 ``[rows]`` (places in the sequence).

        Pages are taken from the stack's top in the sequences' order.  A sequence is refused whose tokens do not fit its
        row of the table, whose rows pass ``rows``, or that lacks pages when the sequences before it have asked for all
        there are; it keeps its length, and its rows, as those past the last, get slot and position -1."""
        return _native.extend(self._address, tokens, rows)

    def truncate(self, lengths) -> None:
        """Shorten sequences to int32 ``lengths`` ``[max_sequences]`` (a longer one changes nothing; 0 or less ends the
        sequence).  Pages past that go back to the stack, the first sequence's first one on top."""
        _native.truncate(self._address, lengths)


def _check_page_size(page_size):
    if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
        raise ValueError(f"page_size must be a power of two from 16 to 1024, got {page_size}")


class _RotaryHandle(ctypes.Structure):  # as csrc/generation_binding.cpp reads it
    _fields_ = [
        ("turns", ctypes.c_void_p),
        ("axes", ctypes.c_void_p),
        ("pairs", ctypes.c_int32),
        ("head_dim", ctypes.c_int32),
        ("neighbours", ctypes.c_int32),
        ("device", ctypes.c_int32),
        ("position_axes", ctypes.c_int32),
    ]


# 1 / (2 pi) to 50 digits.
_PER_TURN = Fraction("0.15915494309189533576888376337251436203445964574046")


class Rotary:
    """Rotary positions with one or several axes (time, height and width of page images, say).

    The first ``rotary_dim`` dimensions of a head (all of ``head_dim`` by default) are ``rotary_dim / 2`` pairs: ``i`` and
    ``rotary_dim / 2 + i`` (``pairs="halves"``) or ``2i`` and ``2i + 1`` (``"neighbours"``).  Pair ``i`` turns by ``position *
    theta ** (-2i / rotary_dim)``, or ``position * frequencies[i]`` where these are given (radians a position).
    ``sections`` says how many pairs go by each axis, one axis by default: consecutive runs, or ``interleaved``, pair
    ``i`` of ``n`` axes by axis ``i % n`` while ``i < n * sections[i % n]`` and by the first one from there.  A
    frequency is a double, held as turns to 2^-64, so that an angle is off by at most ``|position|`` (2^-65 turns and a
    double's rounding of the frequency) before it becomes fp32: less than fp32 shows up to some 10^8 positions."""

    def __init__(self, head_dim, *, sections=None, theta=10000.0, rotary_dim=None, interleaved=False, pairs="halves",
                 frequencies=None, device="cuda"):
        _load()
        head_dim = int(head_dim)
        rotary_dim = head_dim if rotary_dim is None else int(rotary_dim)
        if head_dim < 2 or head_dim > 1024:
            raise ValueError(f"head_dim must be from 2 to 1024, got {head_dim}")
        if rotary_dim < 2 or rotary_dim > head_dim or rotary_dim % 2:
            raise ValueError(f"rotary_dim must be even, from 2 to head_dim, got {rotary_dim}")
        if pairs not in ("halves", "neighbours"):
            raise ValueError(f"pairs must be 'halves' or 'neighbours', got {pairs!r}")
        half = rotary_dim // 2
        sections = [half] if sections is None else [int(n) for n in sections]
        if not sections or min(sections) < 0 or sum(sections) != half or len(sections) > 256:
            raise ValueError(f"sections must be at most 256 numbers of pairs, {half} together, got {sections}")
        n = len(sections)
        if interleaved:
            axes = [i % n if i < n * sections[i % n] else 0 for i in range(half)]
            if [axes.count(a) for a in range(n)] != sections:
                raise ValueError(f"sections {sections} cannot be interleaved over {half} pairs")
        else:
            axes = [a for a, count in enumerate(sections) for _ in range(count)]
        if frequencies is None:
            if not (0.0 < float(theta) < float("inf")):
                raise ValueError("theta must be finite and > 0")
            frequencies = [float(theta) ** (-i / half) for i in range(half)]
        frequencies = [float(f) for f in frequencies]
        if len(frequencies) != half or not all(abs(f) < float("inf") for f in frequencies):
            raise ValueError(f"frequencies must be {half} finite numbers")
        if torch.device(device).type != "cuda":
            raise ValueError(f"Rotary must be on a CUDA device, got {device}")
        turns = [round(Fraction(f) * _PER_TURN * 2**64) % 2**64 for f in frequencies]
        self._turns = torch.tensor([t - 2**64 if t >= 2**63 else t for t in turns], dtype=torch.int64, device=device)
        self._axes = torch.tensor(axes, dtype=torch.uint8, device=device)
        self.device = self._turns.device
        self.head_dim, self.rotary_dim, self.sections = head_dim, rotary_dim, tuple(sections)
        self._c = _RotaryHandle(self._turns.data_ptr(), self._axes.data_ptr(), half, head_dim, pairs == "neighbours",
                                self.device.index, n)
        self._address = ctypes.addressof(self._c)

    def __call__(self, query, keys, positions, *, inverse=False, out=None):
        """``(query, keys)`` ``[tokens, heads, head_dim]`` (fp32, fp16 or bf16, any token and head strides; ``keys`` may
        be None) turned by ``positions`` ``[axes, tokens]`` (int32 or int64; ``[tokens]`` with one axis), ``inverse`` turned
        back.  Products are fp32, rounded once; dimensions past ``rotary_dim`` are copied.  ``out``: a pair of tensors of
        any token and head strides, apart from the inputs, or the inputs themselves."""
        return _native.rotate(self._address, query, keys, positions, inverse, out)


class _Linear(ctypes.Structure):  # as csrc/generation_binding.cpp reads it
    _fields_ = [
        ("codes", ctypes.c_void_p),
        ("scales", ctypes.c_void_p),
        ("bias", ctypes.c_void_p),
        ("n", ctypes.c_int64),
        ("k", ctypes.c_int64),
        ("group", ctypes.c_int32),
        ("bias_type", ctypes.c_int32),
        ("device", ctypes.c_int32),
    ]


class Int4Linear:
    """``x @ W.T + bias`` for few rows ``x`` and weights held as 4-bit codes.

    ``codes`` uint8 ``[out, in / 2]`` (the corpora's nibbles, values -7 to 7) with bfloat16 ``scales`` ``[out,
    ceil(in / group_size)]``; ``group_size`` 32, 64 or 128, ``in`` a multiple of 8.  The weights are laid out once,
    here, for the kernel; ``codes`` and ``scales`` are not kept.  ``bias`` has the dtype of the rows.
    """

    def __init__(self, codes, scales, *, group_size=128, bias=None):
        _load()
        if not hasattr(codes, "data_ptr") or codes.device.type != "cuda":
            raise ValueError("codes must be a CUDA tensor")
        self.device = codes.device
        _on(codes, "codes", self.device, torch.uint8, 2)
        self.out_features, self.in_features = codes.shape[0], 2 * codes.shape[1]
        self.group_size = int(group_size)
        code_bytes, scale_bytes = ctypes.c_int64(), ctypes.c_int64()
        check(lib.msb_w4_packed_bytes(self.out_features, self.in_features, self.group_size, ctypes.byref(code_bytes),
                                      ctypes.byref(scale_bytes)))
        groups = -(-self.in_features // self.group_size)
        _on(scales, "scales", self.device, torch.bfloat16, 2)
        if scales.shape != (self.out_features, groups):
            raise ValueError(f"scales must have shape [{self.out_features}, {groups}], got {list(scales.shape)}")
        if bias is not None:
            _on(bias, "bias", self.device, ndim=1)
            _type_id(bias.dtype, "fp16 or bf16")
            if bias.shape[0] != self.out_features:
                raise ValueError(f"bias must have shape [{self.out_features}]")
            bias = bias.detach().contiguous()
        self._bias = bias
        codes, scales = codes.contiguous(), scales.contiguous()
        with torch.cuda.device(self.device):
            self._codes = torch.empty(code_bytes.value, dtype=torch.uint8, device=self.device)
            self._scales = torch.empty(scale_bytes.value, dtype=torch.uint8, device=self.device)
            check(lib.msb_w4_pack_device(codes.data_ptr(), scales.data_ptr(), self.out_features, self.in_features,
                                         self.group_size, self._codes.data_ptr(), self._scales.data_ptr(),
                                         torch.cuda.current_stream().cuda_stream))
        self._c = _Linear(self._codes.data_ptr(), self._scales.data_ptr(), None if bias is None else bias.data_ptr(),
                          self.out_features, self.in_features, self.group_size,
                          -1 if bias is None else _type_id(bias.dtype, "fp16 or bf16"), self.device.index)
        self._address = ctypes.addressof(self._c)

    @classmethod
    def from_weight(cls, weight, *, group_size=128, bias=None):
        """Quantise ``weight`` ``[out, in]``: per row and group ``scale = bfloat16(max|w| / 7)`` (0 becomes 1),
        ``code = clip(rint(w / scale), -7, 7)`` against the rounded scale."""
        _load()
        if not hasattr(weight, "data_ptr") or weight.dim() != 2:
            raise ValueError("weight must have shape [out, in]")
        if group_size not in (32, 64, 128):
            raise ValueError(f"group_size must be 32, 64 or 128, got {group_size}")
        n, k = weight.shape
        if n < 1 or k < 8 or k % 8:
            raise ValueError("weight must have rows and a multiple of 8 inputs")
        groups = -(-k // group_size)
        w = torch.nn.functional.pad(weight.float(), (0, groups * group_size - k)).view(n, groups, group_size)
        if not torch.isfinite(w).all():
            raise ValueError("weight must contain only finite values")
        scales = (w.abs().amax(dim=2) / 7).to(torch.bfloat16)
        scales[scales == 0] = 1
        codes = torch.round(w / scales.float().unsqueeze(2)).clamp_(-7, 7).to(torch.int16).view(n, -1)[:, :k]
        packed = ((codes[:, 0::2] & 15) | ((codes[:, 1::2] & 15) << 4)).to(torch.uint8)
        return cls(packed, scales, group_size=group_size, bias=bias)

    bias = property(lambda self: self._bias)  # read-only, as its address is held

    @property
    def resident_bytes(self) -> int:
        return self._codes.numel() + self._scales.numel()

    def __call__(self, x, *, out=None):
        """``x`` ``[..., in]`` (fp16 or bf16) to ``[..., out]``; sums are fp32, rounded once.  ``out`` must not overlap
        ``x``."""
        return _native.linear(self._address, x, out)
