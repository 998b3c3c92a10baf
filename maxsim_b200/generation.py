"""Operators of a reader model that answers from retrieved passages, in the codes of the int4 corpora.

``Int4KVCache`` holds keys and values as symmetric 4-bit codes with one fp32 scale per vector (one token, one
head), the layout of a corpus packed as ``int4_per_token``.  Tokens are written as they are produced, read back,
and attended to where they lie.  ``Int4Linear`` multiplies a few rows
with 4-bit weights.  Both take and return CUDA tensors, run on torch's current stream without synchronising,
allocate through torch only, and can be captured into a CUDA graph.

There is no backward pass: these are the operators of serving.  A query or rows that require a gradient are refused
while gradients are enabled; codes, scales and a bias are constants, and keys and values are quantised without one.
"""

from __future__ import annotations

import ctypes

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

    def attend(self, query, page_table, lengths, *, query_offsets=None, max_query_tokens=None, scale=None, causal=True,
               window=None, return_lse=False, out=None):
        """Attention of ``query`` ``[rows, heads, head_dim]`` (fp16 or bf16) over cached tokens.

        ``lengths`` int32 ``[batch]`` counts each sequence's cached tokens, the rows' own among them; int32
        ``page_table`` ``[batch, max_pages]`` names their pages.  Sequence ``b`` owns rows ``query_offsets[b] ..
        query_offsets[b + 1]`` (int32 ``[batch + 1]``, at most ``max_query_tokens`` each), which are its last
        positions; without ``query_offsets`` each sequence has one row.  Rows before the first offset and past the last
        (padding) are zeros, rows past their sequence's ``max_query_tokens`` NaN; a given ``out`` keeps what it holds
        in both (and their log-sum-exp is -inf).  ``max_query_tokens`` defaults to all rows, and the kernel is chosen for
        as many in every sequence: give it where sequences share the rows.

        A row at position ``p`` sees tokens up to ``p`` (``causal``; otherwise all of its sequence), the last
        ``window`` of them where a window is given.  ``heads`` is a multiple of the cache's heads, consecutive
        query heads share one.  ``scale`` defaults to ``head_dim ** -0.5``.  A row that sees nothing is zero.
        Returns ``[rows, heads, head_dim]`` in the query's dtype, with ``return_lse`` also the fp32 natural
        log-sum-exp ``[rows, heads]`` (-inf where nothing is seen), with which results over parts of a context
        can be joined.  ``out`` may be the (contiguous) query itself, but not overlap it otherwise."""
        return _native.attend(self._address, query, page_table, lengths, query_offsets, max_query_tokens, scale, causal,
                              window, return_lse, out)


def _check_cache_sizes(page_size, head_dim):
    if head_dim not in (64, 128, 256):
        raise ValueError(f"head_dim must be 64, 128 or 256, got {head_dim}")
    if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
        raise ValueError(f"page_size must be a power of two from 16 to 1024, got {page_size}")


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
