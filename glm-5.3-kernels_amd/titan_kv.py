# SPDX-License-Identifier: Apache-2.0
"""Per-token symmetric INT8 latent KV writer, MI355X (gfx950) HIP kernel.

Drop-in for `store_int8` of kernels/titan_kv.py:23-28: same name, arguments
and assertions.  The arithmetic runs in the HIP kernel glm53_store_int8
(csrc/store_int8.hip) on the caller's current stream; there is no host sync,
so the call is graph-capturable.

Row format (528 bytes): 512 int8 codes q = clamp(rint(x / s), -127, 127),
fp32 s = max(max|x| / 127, 1e-12) at byte 512, 12 zero bytes.  The quotient
x / s is the correctly rounded IEEE fp32 one.  A negative slot is skipped.

Differences from the reference, all on inputs it leaves undefined:
* a slot at or beyond the cache's capacity (num_blocks * block_size) is
  skipped instead of writing outside the cache;
* the cache may have any 1-byte dtype (it is viewed as int8, as the
  reference does) and its strides are taken in bytes from that view.

Also here: store_rope, the writer of the paged bf16 cache of 576-wide rows
(512 latents, 64 rotated key values; glm53_store_rope, csrc/store_rope.hip),
which titan_mla.mla_chunk_attention_paged reads.
"""
import torch

import _glm53_lib as _lib

_LATENT = 512
_ROW_BYTES = 528


def store_int8(x, cache, slots):
    assert x.shape[-1] == _LATENT and cache.shape[-1] == _ROW_BYTES
    slots = slots.flatten()
    assert slots.numel() <= x.shape[0]
    n = slots.numel()
    if n == 0:
        return
    if not (x.is_cuda and cache.is_cuda and slots.is_cuda):
        raise ValueError("store_int8 requires CUDA (HIP) tensors")
    if x.dtype != torch.bfloat16:
        raise ValueError(f"store_int8 expects bf16 latents, got {x.dtype}")
    if x.stride(-1) != 1:
        x = x.contiguous()
    if slots.dtype not in (torch.int32, torch.int64):
        slots = slots.to(torch.int64)
    slots = slots.contiguous()
    c8 = cache.view(torch.int8)
    block = cache.shape[1]
    capacity = cache.shape[0] * block
    L = _lib.load()
    with torch.cuda.device(x.device):
        rc = L.glm53_store_int8(x.data_ptr(), x.stride(0), c8.data_ptr(), c8.stride(0), c8.stride(1),
                                block, capacity, slots.data_ptr(), int(slots.dtype == torch.int64), n,
                                _lib.stream_handle(x.device))
    _lib.check(rc, "glm53_store_int8")


_ROPE = 64


def _rows16(t):
    """bf16 t where its rows can be read 16 bytes at a time, else a copy."""
    steps = t.stride()
    odd = t.data_ptr() % 16 or steps[-1] != 1
    for step in steps[:-1]:
        odd = odd or step % 8
    return t.clone(memory_format=torch.contiguous_format) if odd else t


def store_rope(x, k_pe, positions, cos_sin, cache, slots, *, q_pe=None, q_out=None, norm_weight=None, eps=1e-6,
               interleaved=False):
    """Append tokens to a paged bf16 latent cache with the position rotation on
    the way: row slots[i] of the cache becomes the latent x[i] (RMS-normed with
    norm_weight, if given) and the rotary key k_pe[i] rotated to positions[i],
    and the queries' rotary parts are rotated with it.  fp32 arithmetic,
    rounded to bf16 once.

    Args:
        x:           bf16 [N, 512] latents
        k_pe:        bf16 [N, 64] rotary keys
        positions:   int32 / int64 [N]
        cos_sin:     fp32 or bf16 [max_pos, 64]: a position's 32 cosines, then
                     its 32 sines
        cache:       bf16 [num_blocks, block_size, 576], strides multiples of 16
                     bytes
        slots:       int32 / int64, at most N of them: token i goes to row
                     slots[i] % block_size of page slots[i] // block_size.  The
                     slots of one call are distinct; a negative one, or one at
                     or past the cache's capacity, is skipped, and tokens behind
                     the last slot are padding (nothing of them is read or
                     written)
        q_pe:        bf16 [N, H, 64] queries' rotary parts, any strides
        q_out:       bf16 [N, H, 64] to write them to, strides multiples of 16
                     bytes - usually q[..., 512:] of the attention's queries
                     (allocated if None; may be q_pe itself)
        norm_weight: bf16 [512]: x is divided by sqrt(mean(x^2) + eps) and
                     multiplied by it
        interleaved: pairs are values (2k, 2k + 1), else (k, 32 + k)

    A token whose position is outside the table leaves its cache row as it
    was, and its queries become zeros.  Returns q_out (None without q_pe).
    """
    # (sizes, strides and addresses are taken once: a small call's time is this function's)
    bf16, xs, ks, cs, ts = torch.bfloat16, x.shape, k_pe.shape, cache.shape, cos_sin.shape
    if len(xs) != 2 or xs[1] != _LATENT or len(ks) != 2 or ks[1] != _ROPE:
        raise ValueError(f"x must be [N, {_LATENT}] and k_pe [N, {_ROPE}], got {tuple(xs)} and {tuple(ks)}")
    if x.dtype is not bf16 or k_pe.dtype is not bf16 or cache.dtype is not bf16:
        raise ValueError("x, k_pe and cache must be bf16")
    page_step, row_step, step = cache.stride() if len(cs) == 3 else (0, 0, 0)
    cache_ptr = cache.data_ptr()
    if step != 1 or cs[2] != _LATENT + _ROPE or page_step % 8 or row_step % 8 or cache_ptr % 16:
        raise ValueError(f"cache must be [num_blocks, block_size, {_LATENT + _ROPE}] with contiguous 16-byte aligned rows")
    table_type = cos_sin.dtype
    if len(ts) != 2 or ts[1] != _ROPE or (table_type is not torch.float32 and table_type is not bf16):
        raise ValueError(f"cos_sin must be fp32 or bf16 [max_pos, {_ROPE}]")
    pos_type, slot_type = positions.dtype, slots.dtype
    pos64, slot64 = pos_type is torch.int64, slot_type is torch.int64
    if not (pos64 or pos_type is torch.int32) or not (slot64 or slot_type is torch.int32):
        raise ValueError(f"positions and slots must be int32 or int64, got {pos_type} and {slot_type}")
    N, n = xs[0], slots.numel()
    if ks[0] != N or positions.numel() != N or n > N:
        raise ValueError(f"{N} latents, {ks[0]} keys, {positions.numel()} positions and {n} slots")
    if norm_weight is not None and (norm_weight.dtype is not bf16 or tuple(norm_weight.shape) != (_LATENT,)):
        raise ValueError(f"norm_weight must be bf16 [{_LATENT}]")
    if q_pe is None and q_out is not None:
        raise ValueError("q_out without q_pe")
    index = x.get_device()
    if index < 0 or k_pe.get_device() != index or positions.get_device() != index or cos_sin.get_device() != index \
            or cache.get_device() != index or slots.get_device() != index \
            or (q_pe is not None and q_pe.get_device() != index) or (q_out is not None and q_out.get_device() != index) \
            or (norm_weight is not None and norm_weight.get_device() != index):
        raise ValueError("store_rope requires CUDA (HIP) tensors on one device")
    heads = sq_t = sq_h = so_t = so_h = 0
    q_ptr = out_ptr = norm_ptr = None
    if q_pe is not None:
        qs = q_pe.shape
        if len(qs) != 3 or qs[0] != N or qs[2] != _ROPE or q_pe.dtype is not bf16:
            raise ValueError(f"q_pe must be bf16 [{N}, H, {_ROPE}], got {q_pe.dtype} {tuple(qs)}")
        if q_out is None:
            q_out = torch.empty((N, qs[1], _ROPE), dtype=bf16, device=x.device)
        so_t, so_h, step = q_out.stride() if q_out.dim() == 3 else (0, 0, 0)
        out_ptr = q_out.data_ptr()
        if q_out.dtype is not bf16 or q_out.shape != qs or step != 1 or so_t % 8 or so_h % 8 or out_ptr % 16:
            raise ValueError(f"q_out must be bf16 {tuple(qs)} with contiguous 16-byte aligned rows")
        q_pe, heads = _rows16(q_pe), qs[1]
        sq_t, sq_h, _ = q_pe.stride()
        q_ptr = q_pe.data_ptr()
    if n == 0:
        return q_out
    x, k_pe = _rows16(x), _rows16(k_pe)
    if not cos_sin.is_contiguous() or cos_sin.data_ptr() % 16:
        cos_sin = cos_sin.clone(memory_format=torch.contiguous_format)
    if norm_weight is not None:
        norm_weight = _rows16(norm_weight)
        norm_ptr = norm_weight.data_ptr()
    positions, slots = positions.contiguous(), slots.contiguous()
    L = _lib.load()
    with _lib.on_device(index):
        rc = L.glm53_store_rope(
            x.data_ptr(), x.stride(0), k_pe.data_ptr(), k_pe.stride(0), positions.data_ptr(), pos64, cos_sin.data_ptr(),
            table_type is torch.float32, ts[0], bool(interleaved), norm_ptr, eps, cache_ptr, 2 * page_step, 2 * row_step,
            max(cs[1], 1), cs[0] * cs[1], slots.data_ptr(), slot64, n, q_ptr, sq_t, sq_h, out_ptr, so_t, so_h, heads,
            _lib.raw_stream(index))
    if rc:
        _lib.check(rc, "glm53_store_rope")
    return q_out
