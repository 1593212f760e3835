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


def _aligned16(t):
    """Whether t's rows can be read 16 bytes at a time: contiguous, every
    other stride and the base a multiple of 16 bytes."""
    size = t.element_size()
    *steps, last = t.stride()
    if last != 1 or t.data_ptr() % 16:
        return False
    for s in steps:
        if s * size % 16:
            return False
    return True


def _rows16(t):
    return t if _aligned16(t) else t.clone(memory_format=torch.contiguous_format)


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
    if x.dim() != 2 or x.shape[1] != _LATENT or k_pe.dim() != 2 or k_pe.shape[1] != _ROPE:
        raise ValueError(f"x must be [N, {_LATENT}] and k_pe [N, {_ROPE}], got {tuple(x.shape)} and {tuple(k_pe.shape)}")
    if x.dtype != torch.bfloat16 or k_pe.dtype != torch.bfloat16 or cache.dtype != torch.bfloat16:
        raise ValueError("x, k_pe and cache must be bf16")
    if cache.dim() != 3 or cache.shape[2] != _LATENT + _ROPE or not _aligned16(cache):
        raise ValueError(f"cache must be [num_blocks, block_size, {_LATENT + _ROPE}] with contiguous 16-byte aligned rows")
    if cos_sin.dim() != 2 or cos_sin.shape[1] != _ROPE or cos_sin.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"cos_sin must be fp32 or bf16 [max_pos, {_ROPE}]")
    for name, t in (("positions", positions), ("slots", slots)):
        if t.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"{name} must be int32 or int64, got {t.dtype}")
    N, n = x.shape[0], slots.numel()
    if k_pe.shape[0] != N or positions.numel() != N or n > N:
        raise ValueError(f"{N} latents, {k_pe.shape[0]} keys, {positions.numel()} positions and {n} slots")
    if norm_weight is not None and (norm_weight.dtype != torch.bfloat16 or tuple(norm_weight.shape) != (_LATENT,)):
        raise ValueError(f"norm_weight must be bf16 [{_LATENT}]")
    if q_pe is None and q_out is not None:
        raise ValueError("q_out without q_pe")
    dev = x.device
    if not x.is_cuda or k_pe.device != dev or positions.device != dev or cos_sin.device != dev \
            or cache.device != dev or slots.device != dev or (q_pe is not None and q_pe.device != dev) \
            or (q_out is not None and q_out.device != dev) or (norm_weight is not None and norm_weight.device != dev):
        raise ValueError("store_rope requires CUDA (HIP) tensors on one device")
    heads = 0
    if q_pe is not None:
        if q_pe.dim() != 3 or q_pe.shape[0] != N or q_pe.shape[2] != _ROPE or q_pe.dtype != torch.bfloat16:
            raise ValueError(f"q_pe must be bf16 [{N}, H, {_ROPE}], got {q_pe.dtype} {tuple(q_pe.shape)}")
        heads = q_pe.shape[1]
        if q_out is None:
            q_out = torch.empty((N, heads, _ROPE), dtype=torch.bfloat16, device=dev)
        elif q_out.dtype != torch.bfloat16 or q_out.shape != q_pe.shape or not _aligned16(q_out):
            raise ValueError(f"q_out must be bf16 {tuple(q_pe.shape)} with contiguous 16-byte aligned rows")
        q_pe = _rows16(q_pe)
    if n == 0:
        return q_out
    x, k_pe = _rows16(x), _rows16(k_pe)
    if not cos_sin.is_contiguous() or cos_sin.data_ptr() % 16:
        cos_sin = cos_sin.clone(memory_format=torch.contiguous_format)
    if norm_weight is not None:
        norm_weight = _rows16(norm_weight)
    positions, slots = positions.contiguous(), slots.contiguous()
    pages, block, _ = cache.shape
    sq_t, sq_h = q_pe.stride()[:2] if heads else (0, 0)
    so_t, so_h = q_out.stride()[:2] if heads else (0, 0)
    L = _lib.load()
    with _lib.on_device(dev):
        rc = L.glm53_store_rope(
            x.data_ptr(), x.stride(0), k_pe.data_ptr(), k_pe.stride(0), positions.data_ptr(),
            positions.dtype == torch.int64, cos_sin.data_ptr(), cos_sin.dtype == torch.float32, cos_sin.shape[0],
            bool(interleaved), norm_weight.data_ptr() if norm_weight is not None else None, eps, cache.data_ptr(),
            2 * cache.stride(0), 2 * cache.stride(1), max(block, 1), pages * block, slots.data_ptr(),
            slots.dtype == torch.int64, n, q_pe.data_ptr() if heads else None, sq_t, sq_h,
            q_out.data_ptr() if heads else None, so_t, so_h, heads, _lib.raw_stream(dev))
    if rc:
        _lib.check(rc, "glm53_store_rope")
    return q_out
