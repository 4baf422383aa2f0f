"""Host-side entry points of the paged key-value cache, the serving side of the attention operator:

* ``page_plan``       — one step of a batch: pages given back and taken, block table, slot map,
* ``paged_append``    — the step's keys and values into the cache (16 bits, or e4m3 with a scale a head),
* ``paged_attention`` — attention of the step's tokens over the pages of their requests.

``syncopate_b200.operators.PagedKVCache`` keeps the state between the steps and calls all three.
Every call goes through the C ABI of ``libsyncopate_b200.so``; none synchronises, so a step can be
captured into a CUDA graph and replayed while the lengths grow.  They read and write device memory
only, on the device of their tensors (which need not be the current one), in the order of ``stream``
(default: that device's current stream).

Index tensors are int32.  What a kernel finds out of range (a length, a page, a slot) it does not
touch; it leaves ``{code, who, value, block}`` in ``status``, a zeroed int32 tensor of four words, with
code 4 (not enough pages) or 5 (index out of range).
"""
from __future__ import annotations

from typing import Optional

import torch

from syncopate_b200 import _lib as L

_DTYPES = {torch.float16: L.SYN_DTYPE_F16, torch.bfloat16: L.SYN_DTYPE_BF16}
HEAD_DIMS = (64, 128, 256)
_INT = torch.int32
_WORKSPACE_BYTES: dict = {}  # (device, num_sms, head dimension) -> bytes


def _refuse(where: str, what: str):
    raise ValueError(f"{where}: {what}")


# Devices are compared by ordinal (-1 = CPU): the calls are made once a layer and token, and a comparison of
# torch.device objects takes several times as long.
def _check_ints(where: str, index: int, **tensors) -> None:
    for name, t in tensors.items():
        if t.dtype is not _INT or t.get_device() != index or not t.is_contiguous():
            _refuse(where, f"{name} must be a contiguous int32 tensor on the device of the others")


def _check_status(where: str, index: int, status) -> int:
    if status is None:
        return 0
    if isinstance(status, int):
        return status
    if status.dtype is not _INT or status.get_device() != index or status.numel() < 4 or not status.is_contiguous():
        _refuse(where, "status must be four int32 words on the device of the others")
    return status.data_ptr()


def _check_table(where: str, index: int, table) -> int:
    """The row stride of a block table."""
    if table.dtype is not _INT or table.get_device() != index or table.dim() != 2:
        _refuse(where, "table must be an int32 [requests, width] tensor on the device of the others")
    rows, width = table.shape
    stride, inner = table.stride()
    if inner != 1 and width > 1:
        _refuse(where, "table must have unit inner stride")
    if stride < width:
        if rows > 1:
            _refuse(where, "the rows of table overlap")
        stride = width  # the stride of a single row says nothing
    return stride


def _stream(device_index: int, stream) -> int:
    if stream is None:
        return torch._C._cuda_getCurrentRawStream(device_index)
    if stream.device_index != device_index:
        raise ValueError(f"stream is on device {stream.device_index}, the tensors are on {device_index}")
    return stream.cuda_stream


def _check_cache(where: str, k_cache, v_cache, dtype, k_scale, v_scale):
    """(cache dtype code, scale pointers) of a pair of caches."""
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape or k_cache.stride() != v_cache.stride():
        _refuse(where, "k_cache and v_cache must be [pages, page_size, heads, dim] with the same shape and strides")
    if k_cache.stride(3) != 1 and k_cache.shape[3] > 1:
        _refuse(where, "the head dimension of the caches must be contiguous")
    kept = k_cache.dtype
    if kept is not v_cache.dtype or k_cache.get_device() != v_cache.get_device():
        _refuse(where, "k_cache and v_cache must agree in type and device")
    if kept is dtype:
        if k_scale is not None or v_scale is not None:
            _refuse(where, "scales belong to an 8-bit cache")
        return L.SYN_CACHE_SAME, 0, 0
    if kept is not torch.float8_e4m3fn:
        _refuse(where, f"the caches must be {dtype} or torch.float8_e4m3fn, not {kept}")
    for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
        if (t is None or t.dtype is not torch.float32 or t.get_device() != k_cache.get_device() or t.dim() != 1
                or t.shape[0] != k_cache.shape[2] or not t.is_contiguous()):
            _refuse(where, f"an 8-bit cache needs {name}, a float32 tensor with one value a head")
    return L.SYN_CACHE_E4M3, k_scale.data_ptr(), v_scale.data_ptr()


def _interleaved(a, b) -> bool:
    """Whether two tensors of one type and shape whose bytes span each other's have no element in common because they
    lie between one another, token by token or head by head, as columns of one projection do."""
    size, shape, sa, sb = a.element_size(), a.shape, a.stride(), b.stride()
    apart, rest = divmod(b.data_ptr() - a.data_ptr(), size)
    if rest:
        return False
    for axis in (0, 1):
        step = sa[axis]
        # All coarser steps are multiples of this one: then what lies within a step decides.
        if step <= 0 or sb[axis] != step or (axis == 1 and shape[0] > 1 and (sa[0] % step or sb[0] % step)):
            continue
        inner_a, inner_b = (1 + sum((n - 1) * s for n, s in zip(shape[axis + 1:], st[axis + 1:])) for st in (sa, sb))
        if apart % step >= inner_a and apart % step + inner_b <= step:
            return True
    return False


def page_plan(
    lens: torch.Tensor,
    add: torch.Tensor,
    table: torch.Tensor,
    free_pages: torch.Tensor,
    num_free: torch.Tensor,
    page_size: int,
    slots: torch.Tensor,
    positions: Optional[torch.Tensor],
    starts: torch.Tensor,
    *,
    lens_out: Optional[torch.Tensor] = None,
    num_free_out: Optional[torch.Tensor] = None,
    status=None,
    stream=None,
) -> None:
    """Plans one step: request ``z`` has ``lens[z]`` cached tokens and appends ``add[z]`` more, or has
    ended (``add[z] < 0``).  ``free_pages[:num_free]`` is a stack; the pages of ended requests are
    pushed onto it, then the new pages popped off it into the rows of ``table``, both in request
    order.  Written: ``slots`` ``[tokens]`` (the step's tokens request by request, -1 behind the last),
    ``positions`` ``[tokens]`` (0 behind the last; may be None), ``starts`` ``[requests + 1]``, and the
    lengths and the number of free pages after the step, in place unless ``lens_out`` /
    ``num_free_out`` are given.  Apart from that no two tensors may overlap.  A step that does not fit
    changes nothing, gives no slots, and is told in ``status``."""
    where = "page_plan"
    index = lens.get_device()
    lens_out = lens if lens_out is None else lens_out
    num_free_out = num_free if num_free_out is None else num_free_out
    table_stride = _check_table(where, index, table)
    _check_ints(where, index, lens=lens, add=add, free_pages=free_pages, num_free=num_free, slots=slots, starts=starts,
                lens_out=lens_out, num_free_out=num_free_out)
    requests, width = table.shape
    if (lens.numel(), add.numel(), starts.numel(), lens_out.numel()) != (requests, requests, requests + 1, requests):
        _refuse(where, "lens, add and lens_out need one entry a row of table, starts one more")
    if num_free.numel() != 1 or num_free_out.numel() != 1:
        _refuse(where, "num_free holds one number")
    if positions is not None:
        _check_ints(where, index, positions=positions)
        if positions.numel() != slots.numel():
            _refuse(where, "positions and slots must have the same length")
    if page_size <= 0:
        _refuse(where, "page_size must be positive")
    if index < 0:
        _refuse(where, "the tensors must be on a CUDA device")
    if requests == 0:
        _refuse(where, "table has no rows")
    args = L.pack_page_plan(
        lens.data_ptr(), add.data_ptr(), table.data_ptr(), free_pages.data_ptr(), num_free.data_ptr(), slots.data_ptr(),
        0 if positions is None else positions.data_ptr(), starts.data_ptr(), lens_out.data_ptr(), num_free_out.data_ptr(),
        _check_status(where, index, status), table_stride, requests, width, page_size, free_pages.numel(),
        slots.numel(), index)
    rc = L.lib().syn_page_plan(args, _stream(index, stream))
    if rc:
        L.check(rc, "syn_page_plan")


def paged_append(
    k: torch.Tensor,
    v: torch.Tensor,
    slots: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    *,
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
    all_slots: bool = False,
    status=None,
    stream=None,
) -> None:
    """Writes row ``t`` of ``k`` and ``v`` ``[tokens, heads, dim]`` to slot ``slots[t]`` of the caches
    ``[pages, page_size, heads, dim]``; negative slots are skipped, ``slots`` may be longer than the rows.  With
    ``all_slots`` what lies behind the rows has to be padding: a slot there that is not negative, a token without a
    row, is told in ``status``.
    The slots of one call must differ from one another: of two rows for one slot parts of both may
    stay.  ``dim`` is a multiple of 16, strides are multiples of 16 bytes, the caches have one layout.
    A ``torch.float8_e4m3fn`` cache keeps ``x / scale[head]`` (float32 division), limited to +-448."""
    where = "paged_append"
    if k.dtype not in _DTYPES or v.dtype is not k.dtype:
        _refuse(where, "k and v must be fp16/bf16 tensors of one type")
    index = k.get_device()
    if k.dim() != 3 or k.shape != v.shape or v.get_device() != index:
        _refuse(where, "k and v must be [tokens, heads, dim] tensors of one shape and device")
    tokens, heads, dim = k.shape
    ks, vs = k.stride(), v.stride()
    if dim > 1 and (ks[2] != 1 or vs[2] != 1):
        _refuse(where, "the head dimension of k and v must be contiguous")
    _check_ints(where, index, slots=slots)
    if slots.numel() < tokens:
        _refuse(where, f"{slots.numel()} slots for {tokens} tokens")
    code, ksp, vsp = _check_cache(where, k_cache, v_cache, k.dtype, k_scale, v_scale)
    pages, page, cache_heads, cache_dim = k_cache.shape
    if (cache_heads, cache_dim) != (heads, dim) or k_cache.get_device() != index:
        _refuse(where, "the caches must be on the device of k and v and have their heads and dim")
    if index < 0:
        _refuse(where, "the tensors must be on a CUDA device")
    num_slots = slots.numel() if all_slots else tokens
    if num_slots == 0:
        return
    cs = k_cache.stride()
    args = L.pack_paged_append(
        k.data_ptr(), v.data_ptr(), slots.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), ksp, vsp,
        _check_status(where, index, status), ks[0], ks[1], vs[0], vs[1], cs[0], cs[1], cs[2], tokens, heads, dim, page, pages,
        _DTYPES[k.dtype], code, index, num_slots)
    rc = L.lib().syn_paged_append(args, _stream(index, stream))
    if rc:
        L.check(rc, "syn_paged_append")


def _workspace(device: torch.device, index: int, num_sms: int, dim: int):
    key = (index, num_sms, dim)
    size = _WORKSPACE_BYTES.get(key)
    if size is None:
        most = torch.cuda.get_device_properties(device).multi_processor_count
        sms = min(num_sms or most, most)
        size = _WORKSPACE_BYTES[key] = L.lib().syn_paged_attention_workspace(sms, dim)
    # From torch's allocator at every call: calls on different streams and captured graphs never share it.
    return torch.empty(size, dtype=torch.uint8, device=device), size


def paged_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    table: torch.Tensor,
    lens: torch.Tensor,
    sm_scale: float,
    *,
    starts: Optional[torch.Tensor] = None,
    causal: bool = True,
    window: int = 0,
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    lse: Optional[torch.Tensor] = None,
    num_sms: int = 0,
    status=None,
    stream=None,
) -> torch.Tensor:
    """``softmax(q k^T * sm_scale) v`` of the newest tokens ``q`` ``[tokens, q_heads, dim]`` over the pages of
    their requests.  Rows ``starts[z]:starts[z + 1]`` (``starts=None``: row ``z`` alone) are the last of the
    ``lens[z]`` tokens that request ``z`` has in the cache, the new ones included, whose pages are
    ``table[z]``.  A row at position ``p`` sees the keys ``j <= p`` (``causal=False``: all of the request's),
    with ``window > 0`` those with ``j > p - window`` only.  ``dim`` is 64, 128 or 256; ``q_heads`` a multiple
    of the caches' heads; the caches hold the type of ``q``, or ``torch.float8_e4m3fn`` with ``k_scale`` and
    ``v_scale`` (what is stored counts times the head's scale).  ``out`` and ``lse`` share no memory with what is
    read; views that lie between the rows or heads of ``q`` (columns of one buffer) are fine.

    ``lse`` ``[tokens, q_heads]`` (float32, optional) receives the log2-sum-exp, with which results over
    parts of a sequence can be joined.  A row that sees no key gives 0 and -inf.  Keys and values that a row
    does not see do not touch it, NaN and infinities included; a value that is not finite and seen leaves its
    dimension not finite (NaN for an infinity too).  Rows behind the last request are left as
    they were (0 where ``out`` is not given).  A row that should see a key without a valid page is NaN.  A
    request with rows behind the end of ``q`` is told in ``status``; its other rows keep their positions.

    The kernel is chosen by the rows of ``q`` a request on average, padding and requests without rows included:
    for decoding pass about as many rows as there are requests (``q[:requests]``), not a buffer for prompts (64
    requests in 512 rows or more: 1.5 times the time, 2.3 times over an 8-bit cache), and a table of the requests
    that are running.

    Scores are meant to stay below 2^29 in magnitude (32 bits leave larger ones no place behind the point).
    Sums, the running maximum and the output are held in 32 bits until the one rounding to ``q``'s type; the
    weights keep 16 bits or more, however small they are, when they meet the values.
    Returns ``out``."""
    where = "paged_attention"
    dtype = q.dtype
    if dtype not in _DTYPES:
        _refuse(where, "q must be an fp16/bf16 tensor")
    if q.dim() != 3:
        _refuse(where, "q must be [tokens, q_heads, dim]")
    index = q.get_device()
    tokens, q_heads, dim = q.shape
    qs = q.stride()
    if qs[2] != 1 or dim not in HEAD_DIMS:
        _refuse(where, f"the head dimension must be contiguous and one of {HEAD_DIMS}")
    code, ksp, vsp = _check_cache(where, k_cache, v_cache, dtype, k_scale, v_scale)
    pages, page, heads, cache_dim = k_cache.shape
    if cache_dim != dim or k_cache.get_device() != index:
        _refuse(where, "the caches must be on the device of q and have its head dimension")
    if heads == 0 or q_heads == 0 or q_heads % heads:
        _refuse(where, f"{q_heads} query heads over {heads} key-value heads")
    table_stride = _check_table(where, index, table)
    _check_ints(where, index, lens=lens)
    requests, width = table.shape
    if lens.numel() != requests:
        _refuse(where, "lens needs one entry a row of table")
    if starts is None:
        if tokens != requests:
            _refuse(where, f"{tokens} rows of q for {requests} requests: pass starts")
    else:
        _check_ints(where, index, starts=starts)
        if starts.numel() != requests + 1:
            _refuse(where, "starts needs one entry more than table has rows")
    if window < 0 or (window and not causal):
        _refuse(where, "window must not be negative and needs causal=True")
    if num_sms < 0:
        _refuse(where, "num_sms must not be negative")
    if out is not None:
        if out.dtype is not dtype or out.shape != q.shape or out.get_device() != index or out.stride(2) != 1:
            _refuse(where, "out must have the shape, type and device of q and a contiguous head dimension")
    if lse is not None and (lse.dtype is not torch.float32 or lse.get_device() != index or lse.shape != q.shape[:2]
                            or not lse.is_contiguous()):
        _refuse(where, "lse must be a contiguous float32 [tokens, q_heads] tensor on the device of q")
    # Warps write rows while others read theirs: what is written may share no byte with what is read.
    cs = k_cache.stride()
    if tokens and (out is not None or lse is not None):
        q_from, k_from, v_from = q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr()
        q_to = q_from + 2 * ((tokens - 1) * qs[0] + (q_heads - 1) * qs[1] + dim)
        held = ((pages - 1) * cs[0] + (page - 1) * cs[1] + (heads - 1) * cs[2] + dim) * (1 if code else 2) if pages and page else 0
        o_from = o_to = 0
        if out is not None:
            os_ = out.stride()
            o_from = out.data_ptr()
            o_to = o_from + 2 * ((tokens - 1) * os_[0] + (q_heads - 1) * os_[1] + dim)
            if q_from < o_to and o_from < q_to and not _interleaved(q, out):
                _refuse(where, "out must not overlap q")
            if k_from < o_to and o_from < k_from + held or v_from < o_to and o_from < v_from + held:
                _refuse(where, "out must not overlap the caches")
        if lse is not None:
            l_from = lse.data_ptr()
            l_to = l_from + 4 * tokens * q_heads
            if (q_from < l_to and l_from < q_to or o_from < l_to and l_from < o_to or k_from < l_to and l_from < k_from + held
                    or v_from < l_to and l_from < v_from + held):
                _refuse(where, "lse must not overlap q, out or the caches")
    if index < 0:
        _refuse(where, "the tensors must be on a CUDA device")
    if stream is not None:
        _stream(index, stream)
        # What is allocated below belongs to the stream that it is used on, and to the device of that stream.
        with torch.cuda.stream(stream):
            return paged_attention(q, k_cache, v_cache, table, lens, sm_scale, starts=starts, causal=causal, window=window,
                                   k_scale=k_scale, v_scale=v_scale, out=out, lse=lse, num_sms=num_sms, status=status)
    if out is None:
        out = (torch.empty if starts is None else torch.zeros)(tokens, q_heads, dim, dtype=dtype, device=q.device)
    if tokens == 0 or requests == 0:
        return out
    os_ = out.stride()
    workspace, size = _workspace(q.device, index, num_sms, dim)
    args = L.pack_paged_attn(
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), table.data_ptr(), lens.data_ptr(),
        0 if starts is None else starts.data_ptr(), out.data_ptr(), 0 if lse is None else lse.data_ptr(), ksp, vsp,
        workspace.data_ptr(), size, _check_status(where, index, status), qs[0], qs[1],
        os_[0], os_[1], cs[0], cs[1], cs[2], table_stride, sm_scale, tokens, requests, q_heads, heads, dim, page,
        pages, width, 1 if causal else 0, window, _DTYPES[dtype], code, num_sms, index)
    rc = L.lib().syn_paged_attention(args, _stream(index, None))
    if rc:
        L.check(rc, "syn_paged_attention")
    return out


__all__ = ["HEAD_DIMS", "page_plan", "paged_append", "paged_attention"]
