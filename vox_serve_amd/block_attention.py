"""Long contexts over a paged cache, on MI355X: new rows rotated into the cache in one call, and attention that reads the blocks of the
context a cheap score picks for each query, not all of it.  Beside the dense operators of `flashinfer_utils` (flashinfer_utils.py:11-324 of the
reference has no sparse form); its wrappers hand their plan to the functions here.

  rope_append      rotate q and k, append k and v at their pages and slots, keep the bounds of completed blocks
  new_bounds       room for the bounds of a cache layer
  update_bounds    the bounds alone, behind another way of filling the cache
  select_blocks    which blocks each row reads
  block_attention  attention over those blocks

A cache layer is [pages, 2, page, kv heads, dim] in bf16 or fp16, dim 64 or 128, a page whole blocks of 16, 32, 64 or 128 tokens.  `bounds`
(int8 [pages, kv heads, blocks a page, 2, dim]) holds the largest and the smallest key of a complete block per channel, as whole numbers of
`steps` (fp32 [pages, kv heads, blocks a page], powers of two).  Integer plan arrays are int32 (int64 is converted, its
values have to fit).  Rows whose page is negative, or that see no token, are passed over: what would have been written for them stays as it was.
"""
import functools
import struct

import torch

from . import _native as N

_DTYPES = {torch.bfloat16: 0, torch.float16: 1}
_CACHE = "PPP6i"
_ROWS = "PPPP6i"                        # (the last one pads to eight bytes)
_APPEND = struct.Struct(_CACHE + "PPPPPPPP3q6i")
_BOUNDS = struct.Struct(_CACHE)
_SELECT = struct.Struct(_CACHE + _ROWS + "PPP2q3i0q")
_ATTEND = struct.Struct(_CACHE + _ROWS + "PPPP2qif0q")


def _on(device):
    """Context and stream of the device that is current.  (The raw stream costs 0.1 us, a torch.cuda.Stream object of it 2.7: as much as the launch.)"""
    return N._ctxs.get(device.index) or N.ctx(), torch._C._cuda_getCurrentRawStream(device.index)


@functools.lru_cache(maxsize=4096)
def _attend_room(*sizes):
    """Bytes of workspace that a call of these sizes asks for: a function of the sizes alone."""
    rows, n_own, heads, kv_heads, dim, dtype, page, block, top = sizes
    n = N.lib().vox_block_attention_workspace_bytes(_ATTEND.pack(16, 0, 0, 1, page, block, kv_heads, dim, dtype, 16, 16, 16, 16, rows, 1, n_own, heads, 1, 0, 16, 16, 16, 0, 0, 0, top, 1.0))
    return max(n, 0)                    # (sizes that the call itself will refuse)


@functools.lru_cache(maxsize=4096)
def _select_room(*sizes):
    rows, n_own, heads, kv_heads, dim, dtype, page, block, top, first, last, max_kvlen = sizes
    n = N.lib().vox_block_select_workspace_bytes(_SELECT.pack(0, 16, 16, 1, page, block, kv_heads, dim, dtype, 16, 16, 16, 16, rows, 1, n_own, heads, max_kvlen, 0, 16, 16, 0, 0, 0, top, first, last))
    return max(n, 0)


def _device(t, name):
    d = t.device
    if d.type != "cuda":
        raise ValueError(f"{name} is on {d}: libvoxhip takes tensors of a HIP device")
    return d


def _ints(t, shape, device, name):
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, {tuple(shape)} is wanted")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the cache on {device}")
    if t.dtype is not torch.int32:
        if t.dtype is not torch.int64:
            raise TypeError(f"{name} is {t.dtype}: int32 or int64 is wanted")
        t = N.hold(t.to(torch.int32))
    return t if t.is_contiguous() else N.hold(t.contiguous())


def _heads(t, rows, dim, like, name):
    """[rows, heads, dim] whose heads lie together; rows may lie apart."""
    shape = t.shape
    if len(shape) != 3 or shape[0] != rows or shape[2] != dim:
        raise ValueError(f"{name} has shape {tuple(shape)}, [{rows}, heads, {dim}] is wanted")
    if t.dtype is not like.dtype or t.device != like.device:
        raise ValueError(f"{name} is {t.dtype} on {t.device}, {like.dtype} on {like.device} is wanted")
    _, apart, unit = t.stride()
    return t if unit == 1 and (apart == dim or shape[1] == 1) else N.hold(t.contiguous())


def _cache(kv):
    if kv.dim() != 5 or kv.shape[1] != 2 or not kv.is_contiguous():
        raise ValueError(f"kv_cache has shape {tuple(kv.shape)}: a contiguous [pages, 2, page, kv heads, dim] is wanted")
    if kv.dtype not in _DTYPES:
        raise TypeError(f"kv_cache is {kv.dtype}: bfloat16 or float16 is wanted")
    return _device(kv, "kv_cache")


def _bounds(bounds, steps, device):
    """The shape (pages, kv heads, blocks, 2, dim)."""
    shape = bounds.shape
    if len(shape) != 5 or shape[3] != 2 or bounds.dtype is not torch.int8 or not bounds.is_contiguous():
        raise ValueError(f"bounds is {bounds.dtype} {tuple(shape)}: a contiguous int8 [pages, kv heads, blocks, 2, dim] is wanted")
    if steps.shape != shape[:3] or steps.dtype is not torch.float32 or not steps.is_contiguous():
        raise ValueError(f"steps is {steps.dtype} {tuple(steps.shape)}: a contiguous float32 {tuple(shape[:3])} is wanted")
    if bounds.device != device or steps.device != device:
        raise ValueError(f"bounds and steps are on {bounds.device} and {steps.device}, {device} is wanted")
    return shape


def _bounds_of(kv, bounds, steps):
    """(bounds, steps, block) of a cache layer, as pointers."""
    if bounds is None or steps is None:
        raise ValueError("bounds and steps come together")
    pages, heads, per, _, dim = _bounds(bounds, steps, kv.device)
    p, _, page, h, d = kv.shape
    if pages != p or heads != h or dim != d or per == 0 or page % per:
        raise ValueError(f"bounds {tuple(bounds.shape)} are not those of a cache {tuple(kv.shape)}")
    return bounds.data_ptr(), steps.data_ptr(), page // per


def _out(out, shape, like, device, name="out"):
    if out is None:
        return N.hold(torch.empty(shape, dtype=like, device=device))      # (rows that are passed over hold what the allocator left)
    if out.shape != shape or out.dtype is not like or out.device != device or not out.is_contiguous():
        raise ValueError(f"{name} is {out.dtype} {tuple(out.shape)} on {out.device}: a contiguous {like} {tuple(shape)} on {device} is wanted")
    return out


def new_bounds(kv_cache, block):
    """(bounds, steps) for a cache layer whose pages are cut into blocks of `block` tokens: zero until rows complete blocks."""
    p, _, page, h, d = kv_cache.shape
    if block <= 0 or page % block:
        raise ValueError(f"pages of {page} tokens are not whole blocks of {block}")
    return (torch.zeros(p, h, page // block, 2, d, dtype=torch.int8, device=kv_cache.device),
            torch.zeros(p, h, page // block, dtype=torch.float32, device=kv_cache.device))


def rope_append(q, k, v, kv_cache, cos_sin, positions, pages, slots, *, interleave=False, bounds=None, steps=None, n_req=0, out=None):
    """Rotate q [rows, heads, dim] and k [rows, kv heads, dim] by their rows' positions and append k and v to the cache at (pages, slots).
    Returns the rotated q (`out` if it is given; q itself serves if it is contiguous).

    q, k and v may be slices of one projection's output.  cos_sin: fp32 [positions, channels that turn / 2, 2] (`flashinfer_utils.rope_table`:
    plain, scaled and llama-3.1 angles; fewer channels than dim: the others stay), or None: nothing turns.  Positions are clamped to the table.
    By the same table the results are those of `apply_rope_pos_ids` (whose own has 8192 positions) and `set_kv_cache`, bit for bit.  With `bounds`
    and `steps` (`new_bounds`), also those of the blocks that the rows complete, by their last token (behind a row that overwrites an earlier one:
    `update_bounds` with that block's last slot).  n_req: how many requests have rows here, 0 if it is not known; as many as rows: a token of
    each, one launch."""
    device = _cache(kv_cache)
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return rope_append(q, k, v, kv_cache, cos_sin, positions, pages, slots, interleave=interleave, bounds=bounds, steps=steps, n_req=n_req, out=out)
    n_pages, _, page, h, d = kv_cache.shape
    rows = q.shape[0]
    q, k, v = _heads(q, rows, d, kv_cache, "q"), _heads(k, rows, d, kv_cache, "k"), _heads(v, rows, d, kv_cache, "v")
    if k.shape[1] != h or v.shape[1] != h:
        raise ValueError(f"k and v have {k.shape[1]} and {v.shape[1]} heads, the cache {h}")
    one = (rows,)
    positions, pages, slots = _ints(positions, one, device, "positions"), _ints(pages, one, device, "pages"), _ints(slots, one, device, "slots")
    rot, table, length = 0, 0, 0
    if cos_sin is not None:
        if cos_sin.dim() != 3 or cos_sin.shape[2] != 2 or cos_sin.dtype is not torch.float32 or cos_sin.device != device:
            raise ValueError(f"cos_sin is {cos_sin.dtype} {tuple(cos_sin.shape)} on {cos_sin.device}: float32 [positions, turning channels / 2, 2] on {device} is wanted")
        cos_sin = cos_sin if cos_sin.is_contiguous() else N.hold(cos_sin.contiguous())
        rot, table, length = 2 * cos_sin.shape[1], cos_sin.data_ptr(), cos_sin.shape[0]
    where = (0, 0, page) if bounds is None and steps is None else _bounds_of(kv_cache, bounds, steps)
    out = _out(out, q.shape, kv_cache.dtype, device)
    ctx, stream = _on(device)
    N.check(N.lib().vox_rope_append(ctx, stream, _APPEND.pack(
        kv_cache.data_ptr(), where[0], where[1], n_pages, page, where[2], h, d, _DTYPES[kv_cache.dtype], q.data_ptr(), k.data_ptr(), v.data_ptr(),
        out.data_ptr(), positions.data_ptr(), pages.data_ptr(), slots.data_ptr(), table, q.stride(0), k.stride(0), v.stride(0), rows, n_req, q.shape[1], rot,
        1 if interleave else 0, length)))
    return out


def update_bounds(kv_cache, bounds, steps, pages, slots):
    """The bounds of the blocks whose last token is at one of (pages, slots): what `rope_append` keeps by itself, behind another way of
    filling the cache."""
    device = _cache(kv_cache)
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return update_bounds(kv_cache, bounds, steps, pages, slots)
    n_pages, _, page, h, d = kv_cache.shape
    one = (pages.shape[0],)
    pages, slots = _ints(pages, one, device, "pages"), _ints(slots, one, device, "slots")
    where = _bounds_of(kv_cache, bounds, steps)
    ctx, stream = _on(device)
    N.check(N.lib().vox_block_bounds(ctx, stream, _BOUNDS.pack(kv_cache.data_ptr(), where[0], where[1], n_pages, page, where[2], h, d, _DTYPES[kv_cache.dtype]),
                                     pages.data_ptr(), slots.data_ptr(), one[0]))


def _plan(q_req, q_kvlen, kv_indptr, kv_indices, rows, device):
    one = (rows,)
    return (_ints(q_req, one, device, "q_req"), _ints(q_kvlen, one, device, "q_kvlen"), _ints(kv_indptr, kv_indptr.shape[:1], device, "kv_indptr"),
            _ints(kv_indices, kv_indices.shape[:1], device, "kv_indices"))


def select_blocks(q, bounds, steps, q_req, q_kvlen, kv_indptr, kv_indices, *, block, top, max_kvlen, first=1, last=2, n_req=0, out=None):
    """The blocks that each row reads: int32 [rows, kv heads, top], ascending, -1 behind the last.

    A row of n tokens has ceil(n / block) blocks.  Its first `first` and its newest `last` (at least one) are always among them; the others
    are those with the largest bound on the sum of a kv head's q . k, taken from 8-bit `bounds` and q rounded to 8 bits - whole numbers, so the choice does not
    depend on batch or launch -, the older one where bounds are equal.  q [rows, heads, dim], rotated; max_kvlen: no row sees more tokens."""
    device = _device(bounds, "bounds")
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return select_blocks(q, bounds, steps, q_req, q_kvlen, kv_indptr, kv_indices, block=block, top=top, max_kvlen=max_kvlen, first=first, last=last, n_req=n_req, out=out)
    n_pages, h, per, _, d = _bounds(bounds, steps, device)
    rows = q.shape[0]
    if q.dtype not in _DTYPES:
        raise TypeError(f"q is {q.dtype}: bfloat16 or float16 is wanted")
    if q.device != device:
        raise ValueError(f"q is on {q.device}, the bounds on {device}")
    q = _heads(q, rows, d, q, "q")
    plan = _plan(q_req, q_kvlen, kv_indptr, kv_indices, rows, device)
    out = _out(out, (rows, h, top), torch.int32, device)
    room = _select_room(rows, n_req, q.shape[1], h, d, _DTYPES[q.dtype], per * block, block, top, first, last, max_kvlen)
    ws = N.hold(torch.empty(room, dtype=torch.uint8, device=device)) if room else None
    ctx, stream = _on(device)
    N.check(N.lib().vox_block_select(ctx, stream, _SELECT.pack(
        0, bounds.data_ptr(), steps.data_ptr(), n_pages, per * block, block, h, d, _DTYPES[q.dtype], plan[0].data_ptr(), plan[1].data_ptr(), plan[2].data_ptr(),
        plan[3].data_ptr(), rows, plan[2].shape[0] - 1, n_req, q.shape[1], max_kvlen, 0, q.data_ptr(), out.data_ptr(),
        ws.data_ptr() if room else 0, room, q.stride(0), top, first, last)))
    return out


def block_attention(q, kv_cache, blocks, q_req, q_kvlen, kv_indptr, kv_indices, *, block, scale=None, n_req=0, out=None):
    """softmax(scale q . K) V over the tokens that a row sees (its first q_kvlen) of the blocks in its lists, int32 [rows, kv heads, top] as of `select_blocks`.

    An entry counts if it is a block of the row and larger than the entries before it; a row without any is zero.  scale: 1 / sqrt(dim) if
    it is not given.  n_req: how many requests have rows here, 0 if it is not known.  Sizes and n_req choose the launch, and by that the order of a
    row's fp32 sums; what the tokens of other rows hold changes nothing, not a bit."""
    device = _cache(kv_cache)
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return block_attention(q, kv_cache, blocks, q_req, q_kvlen, kv_indptr, kv_indices, block=block, scale=scale, n_req=n_req, out=out)
    n_pages, _, page, h, d = kv_cache.shape
    rows = q.shape[0]
    q = _heads(q, rows, d, kv_cache, "q")
    if blocks.dim() != 3:
        raise ValueError(f"blocks has shape {tuple(blocks.shape)}, [{rows}, {h}, top] is wanted")
    top = blocks.shape[2]
    blocks = _ints(blocks, (rows, h, top), device, "blocks")
    plan = _plan(q_req, q_kvlen, kv_indptr, kv_indices, rows, device)
    out = _out(out, q.shape, kv_cache.dtype, device)
    ctx, stream = _on(device)
    room = _attend_room(rows, n_req, q.shape[1], h, d, _DTYPES[kv_cache.dtype], page, block, top)
    ws = N.hold(torch.empty(room, dtype=torch.uint8, device=device)) if room else None
    N.check(N.lib().vox_block_attention(ctx, stream, _ATTEND.pack(
        kv_cache.data_ptr(), 0, 0, n_pages, page, block, h, d, _DTYPES[kv_cache.dtype], plan[0].data_ptr(), plan[1].data_ptr(), plan[2].data_ptr(),
        plan[3].data_ptr(), rows, plan[2].shape[0] - 1, n_req, q.shape[1], 2 ** 31 - 1, 0, q.data_ptr(), blocks.data_ptr(), out.data_ptr(),
        ws.data_ptr() if room else 0, room, q.stride(0), top, d ** -0.5 if scale is None else scale)))
    return out
