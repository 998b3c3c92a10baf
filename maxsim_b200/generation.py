"""Operators of a reader model that answers from retrieved passages, in the codes of the int4 corpora.

``Int4KVCache`` holds keys and values as symmetric 4-bit codes with one fp32 scale per vector (one token, one
head), the layout of a corpus packed as ``int4_per_token``.  Tokens are written as they are produced, read back,
and attended to where they lie.  ``Int4Linear`` multiplies a few rows
with 4-bit weights.  Both take and return CUDA tensors, run on torch's current stream without synchronising,
allocate through torch only, and can be captured into a CUDA graph.

There is no backward pass: codes have no gradient, and these are the operators of serving.
"""

from __future__ import annotations

import ctypes
import math

torch = _lib = lib = check = None


def _load():
    """Import torch and the CUDA library, once, when the first object is made (the package imports without them)."""
    global torch, _lib, lib, check
    if _lib is None:
        import torch as torch_module
        from maxsim_b200 import _lib as lib_module

        torch, lib, check = torch_module, lib_module.lib, lib_module.check
        _lib = lib_module


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
        """A cache over arrays the caller owns (shapes above, contiguous)."""
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
        self.k_codes, self.k_scales, self.v_codes, self.v_scales = k_codes, k_scales, v_codes, v_scales
        self.device = device
        self.num_pages, self.num_kv_heads, self.page_size, self.head_dim = pages, heads, size, 2 * half
        self._c = _lib.Kv4Cache(k_codes.data_ptr(), k_scales.data_ptr(), v_codes.data_ptr(), v_scales.data_ptr(), pages,
                                size, heads, 2 * half, device.index)
        self._ref = ctypes.byref(self._c)

    @property
    def resident_bytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k_codes, self.k_scales, self.v_codes, self.v_scales))

    def _stream(self):
        return torch.cuda.current_stream(self.device).cuda_stream

    def _vectors(self, x, name, tokens=None):
        _on(x, name, self.device, ndim=3)
        if x.shape[1] != self.num_kv_heads or x.shape[2] != self.head_dim:
            raise ValueError(f"{name} must have shape [tokens, {self.num_kv_heads}, {self.head_dim}], got {list(x.shape)}")
        if tokens is not None and x.shape[0] != tokens:
            raise ValueError("keys, values and slots must have the same number of tokens")
        return x if x.stride(2) == 1 else x.contiguous()

    def _slots(self, slots):
        _on(slots, "slots", self.device, torch.int64, 1)
        return slots if slots.is_contiguous() else slots.contiguous()

    def append(self, keys, values, slots) -> None:
        """Quantise ``keys`` and ``values`` ``[tokens, kv_heads, head_dim]`` (fp32, fp16 or bf16, any token and
        head strides) into int64 ``slots`` ``[tokens]``.

        Per vector: ``scale = max|x| * fl(1/7)`` (0 becomes 1), ``code = clip(rint(x / scale), -7, 7)``.  A vector with
        a value that is not finite stores scale NaN and codes 0.  A slot outside the cache (-1, say) is skipped; a
        slot must not be given twice in one call."""
        slots = self._slots(slots)
        tokens = slots.shape[0]
        keys, values = self._vectors(keys, "keys", tokens), self._vectors(values, "values", tokens)
        if keys.dtype != values.dtype:
            raise ValueError("keys and values must have the same dtype")
        check(lib.msb_kv4_append_device(self._ref, keys.data_ptr(), values.data_ptr(), _type_id(keys.dtype), tokens,
                                        keys.stride(0), keys.stride(1), values.stride(0), values.stride(1),
                                        slots.data_ptr(), self._stream()))

    def read(self, slots, *, dtype=None, out=None):
        """``(keys, values)`` of int64 ``slots`` as ``[tokens, kv_heads, head_dim]`` of ``dtype`` (bf16 by default):
        ``code * scale`` rounded once; zeros for a slot outside the cache.  ``out``: a pair of contiguous tensors."""
        slots = self._slots(slots)
        shape = (slots.shape[0], self.num_kv_heads, self.head_dim)
        if out is None:
            dtype = torch.bfloat16 if dtype is None else dtype
            kind = _type_id(dtype)
            out = (torch.empty(shape, dtype=dtype, device=self.device), torch.empty(shape, dtype=dtype, device=self.device))
        else:
            kind = _type_id(out[0].dtype)
            if dtype is not None and dtype != out[0].dtype:
                raise ValueError("out must have the given dtype")
            for name, t in zip(("out[0]", "out[1]"), out):
                _on(t, name, self.device, out[0].dtype)
                if t.shape != shape or not t.is_contiguous():
                    raise ValueError(f"{name} must be contiguous with shape {list(shape)}")
                if t.data_ptr() % 16:
                    raise ValueError(f"{name} must be 16-byte aligned")
        check(lib.msb_kv4_read_device(self._ref, slots.data_ptr(), shape[0], kind, out[0].data_ptr(), out[1].data_ptr(),
                                      self._stream()))
        return tuple(out)

    def slots(self, page_table, sequences, positions):
        """int64 slots of ``positions`` of ``sequences`` (tensors of one shape) under ``page_table``."""
        positions = positions.long()
        return page_table[sequences.long(), positions // self.page_size].long() * self.page_size + positions % self.page_size

    def attend(self, query, page_table, lengths, *, query_offsets=None, max_query_tokens=None, scale=None, causal=True,
               window=None, return_lse=False, out=None):
        """Attention of ``query`` ``[rows, heads, head_dim]`` (fp16 or bf16) over cached tokens.

        ``lengths`` int32 ``[batch]`` counts each sequence's cached tokens, the rows' own among them; int32
        ``page_table`` ``[batch, max_pages]`` names their pages.  Sequence ``b`` owns rows ``query_offsets[b] ..
        query_offsets[b + 1]`` (int32 ``[batch + 1]``, at most ``max_query_tokens`` each), which are its last
        positions; without ``query_offsets`` each sequence has one row.  Every row must belong to a sequence:
        others are not written.

        A row at position ``p`` sees tokens up to ``p`` (``causal``; otherwise all of its sequence), the last
        ``window`` of them where a window is given.  ``heads`` is a multiple of the cache's heads, consecutive
        query heads share one.  ``scale`` defaults to ``head_dim ** -0.5``.  A row that sees nothing is zero.
        Returns ``[rows, heads, head_dim]`` in the query's dtype, with ``return_lse`` also the fp32 natural
        log-sum-exp ``[rows, heads]`` (-inf where nothing is seen), with which results over parts of a context
        can be joined."""
        device = self.device
        _on(query, "query", device, ndim=3)
        kind = _type_id(query.dtype, "fp16 or bf16")
        rows, heads, dim = query.shape
        if dim != self.head_dim or heads == 0 or heads % self.num_kv_heads:
            raise ValueError(f"query must have shape [rows, a multiple of {self.num_kv_heads}, {self.head_dim}], got "
                             f"{list(query.shape)}")
        if query.stride(2) != 1:
            query = query.contiguous()
        _on(page_table, "page_table", device, torch.int32, 2)
        _on(lengths, "lengths", device, torch.int32, 1)
        batch, pages = page_table.shape
        if lengths.shape[0] != batch:
            raise ValueError("page_table and lengths must have the same batch")
        if pages > 1 and page_table.stride(1) != 1:
            page_table = page_table.contiguous()
        if not lengths.is_contiguous():
            lengths = lengths.contiguous()
        if query_offsets is None:
            if rows != batch:
                raise ValueError("without query_offsets, query must have one row per sequence")
            if max_query_tokens not in (None, 1):
                raise ValueError("max_query_tokens needs query_offsets")
            most = 1
        else:
            _on(query_offsets, "query_offsets", device, torch.int32, 1)
            if query_offsets.shape[0] != batch + 1:
                raise ValueError("query_offsets must have shape [batch + 1]")
            if not query_offsets.is_contiguous():
                query_offsets = query_offsets.contiguous()
            most = rows if max_query_tokens is None else int(max_query_tokens)
            if most < 0:
                raise ValueError("max_query_tokens must not be negative")
        if window is not None and (int(window) < 1 or not causal):
            raise ValueError("window must be at least 1 and needs causal")
        scale = dim ** -0.5 if scale is None else float(scale)
        if not (scale > 0.0 and math.isfinite(scale)):
            raise ValueError("scale must be finite and > 0")
        shape = (rows, heads, dim)
        if out is None:
            out = torch.empty(shape, dtype=query.dtype, device=device)
        else:
            _on(out, "out", device, query.dtype)
            if out.shape != shape or not out.is_contiguous():
                raise ValueError(f"out must be contiguous with shape {list(shape)}")
        lse = torch.empty((rows, heads), dtype=torch.float32, device=device) if return_lse else None
        args = _lib.Kv4AttendArgs(
            query.data_ptr(), query.stride(0), query.stride(1), rows, page_table.data_ptr(), page_table.stride(0),
            lengths.data_ptr(), None if query_offsets is None else query_offsets.data_ptr(), out.data_ptr(),
            None if lse is None else lse.data_ptr(), None, 0, batch, pages, most, heads, kind, 1 if causal else 0,
            int(window or 0), scale)
        ref = ctypes.byref(args)
        need = ctypes.c_int64()
        check(lib.msb_kv4_attend_workspace_bytes(self._ref, ref, ctypes.byref(need)))
        if need.value:
            workspace = torch.empty(need.value, dtype=torch.uint8, device=device)
            args.workspace, args.workspace_bytes = workspace.data_ptr(), need.value
        check(lib.msb_kv4_attend_device(self._ref, ref, self._stream()))
        return (out, lse) if return_lse else out


def _check_cache_sizes(page_size, head_dim):
    if head_dim not in (64, 128, 256):
        raise ValueError(f"head_dim must be 64, 128 or 256, got {head_dim}")
    if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
        raise ValueError(f"page_size must be a power of two from 16 to 1024, got {page_size}")


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
            bias = bias.contiguous()
        self.bias = bias
        codes, scales = codes.contiguous(), scales.contiguous()
        with torch.cuda.device(self.device):
            self._codes = torch.empty(code_bytes.value, dtype=torch.uint8, device=self.device)
            self._scales = torch.empty(scale_bytes.value, dtype=torch.uint8, device=self.device)
            check(lib.msb_w4_pack_device(codes.data_ptr(), scales.data_ptr(), self.out_features, self.in_features,
                                         self.group_size, self._codes.data_ptr(), self._scales.data_ptr(),
                                         torch.cuda.current_stream().cuda_stream))

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

    @property
    def resident_bytes(self) -> int:
        return self._codes.numel() + self._scales.numel()

    def __call__(self, x, *, out=None):
        """``x`` ``[..., in]`` (fp16 or bf16) to ``[..., out]``; sums are fp32, rounded once."""
        _on(x, "x", self.device)
        kind = _type_id(x.dtype, "fp16 or bf16")
        if x.dim() < 1 or x.shape[-1] != self.in_features:
            raise ValueError(f"x must have shape [..., {self.in_features}], got {list(x.shape)}")
        if self.bias is not None and self.bias.dtype != x.dtype:
            raise ValueError("bias and x must have the same dtype")
        lead = x.shape[:-1]
        rows = x if x.dim() == 2 else x.reshape(-1, self.in_features)
        if rows.stride(1) != 1:
            rows = rows.contiguous()
        if out is None:
            out = torch.empty(lead + (self.out_features,), dtype=x.dtype, device=self.device)
        else:
            _on(out, "out", self.device, x.dtype)
            if out.shape != lead + (self.out_features,) or not out.is_contiguous():
                raise ValueError(f"out must be contiguous with shape {list(lead) + [self.out_features]}")
        check(lib.msb_w4_product_device(
            self._codes.data_ptr(), self._scales.data_ptr(), self.out_features, self.in_features, self.group_size,
            rows.data_ptr(), rows.stride(0), rows.shape[0], None if self.bias is None else self.bias.data_ptr(),
            out.data_ptr(), self.out_features, kind, self.device.index,
            torch.cuda.current_stream(self.device).cuda_stream))
        return out
