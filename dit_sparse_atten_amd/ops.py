"""Torch-facing wrappers over the libdsa C-ABI.

Tensors are only plumbing here: device memory and the current HIP stream are
taken from PyTorch and passed as raw pointers.  Every compute call runs a
hand-written HIP kernel; there is no CPU or PyTorch fallback, and a CPU tensor
is rejected with ``ValueError``.
"""

from __future__ import annotations

import ctypes
import functools
import math
import typing

import torch

from . import _lib

HEAD_DIM = 128
# Per-row statistics (8 bytes each) that a routed tile call takes room for
# without reading how many its route lists: 256 MiB.  At 1,024 tokens x 12 heads
# the read kept the host behind the device: a step 116 us with it, 83 without.
MAX_UNCOUNTED_ROWS = 1 << 25


def _stream_handle(device) -> int:
    # The handle without a Stream object around it: the three calls of a short
    # route update (512 to 2,400 tokens) are bound by the host, 42 us with the
    # object and 35 without.  A tensor's device always has an index.
    return torch._C._cuda_getCurrentRawStream(device.index)


def _require_cuda(name, tensor):
    if not isinstance(tensor, torch.Tensor) or not tensor.is_cuda:
        raise ValueError(f"{name} must be a CUDA (HIP) tensor; libdsa has no CPU path")


# The 16-bit element types every kernel computes in (dtype codes of dsa.h).
KERNEL_DTYPES = {torch.bfloat16: _lib.DSA_DTYPE_BF16, torch.float16: _lib.DSA_DTYPE_F16}
# The attention (bsa_fwd, bsa_fwd_tile_stats) also computes in float32.
ATTENTION_DTYPES = {**KERNEL_DTYPES, torch.float32: _lib.DSA_DTYPE_F32}


def dtype_code(dtype, attention=False):
    """The libdsa dtype code of a torch dtype; ValueError for any other than
    bfloat16 and float16, or also float32 for the attention
    (``attention=True``)."""
    table = ATTENTION_DTYPES if attention else KERNEL_DTYPES
    if dtype not in table:
        kinds = "bfloat16, float16 or float32" if attention else "bfloat16 or float16"
        raise ValueError(f"libdsa computes in {kinds} here, not {dtype}")
    return table[dtype]


def _kernel_view(name, tensor, dtype=None, attention=False):
    """Return a [B,T,H,D] view the kernel can read (copying only if needed);
    ``dtype``, when given, is the element type every operand must share."""
    _require_cuda(name, tensor)
    if tensor.ndim != 4:
        raise ValueError(f"{name} must have shape [batch, tokens, heads, head_dim]")
    dtype_code(tensor.dtype, attention)
    if dtype is not None and tensor.dtype != dtype:
        raise ValueError(f"{name} must be {dtype} like q, got {tensor.dtype}")
    ok = (
        tensor.stride(3) == 1
        and all(stride % 8 == 0 for stride in tensor.stride()[:3])
        and tensor.data_ptr() % 16 == 0
    )
    return tensor if ok else tensor.contiguous()


def _smaller_workspace(device, *sizes):
    """A workspace of the first of ``sizes`` (descending; 0: None) that the device
    has memory for, of a call that has another way with it."""
    for index, size in enumerate(sizes):
        try:
            return torch.empty(size, dtype=torch.uint8, device=device) if size else None
        except torch.OutOfMemoryError:
            if index + 1 == len(sizes):
                raise


def _f32_workspace_bytes(lib, q, batch, heads, kv_tokens, head_dim, block_size, every_key):
    """Workspace of the float32 attention's split products (0 for the 16-bit
    types, for few keys, for head dims above 128, and below 64 unless every row
    attends every key)."""
    if q.dtype != torch.float32 or (head_dim < 64 and not every_key):
        return 0
    return lib.dsa_bsa_f32_workspace_bytes_block(batch, heads, kv_tokens, head_dim, block_size)


def _statistics_workspace_bytes(lib, q, own, heads, tokens, head_dim, block_size, dense):
    """Workspace of an attention call with statistics: ``own`` bytes, in which
    the float32 split products take the place of the 16-bit kernels' scratch."""
    more = _f32_workspace_bytes(lib, q, 1, heads, tokens, head_dim, block_size, dense)
    if more:
        own += max(0, more - lib.dsa_bsa_workspace_bytes_block(1, heads, tokens, head_dim,
                                                               block_size))
    return own


class RouteCSR:
    """Compressed block route: for every (route batch, head, query block) row,
    the ascending list of key blocks it attends to.

    This is the MI355X counterpart of the KV half of a FlexAttention
    ``BlockMask`` (``full_kv_num_blocks`` / ``full_kv_indices``,
    attention_backends/flex.py:326-338), keeping only the selected prefix.
    """

    __slots__ = ("row_ptr", "col_idx", "counts", "route_batches", "heads",
                 "q_blocks", "k_blocks", "block_size", "nnz", "_route")

    def __init__(self, row_ptr, col_idx, counts, route_batches, heads, q_blocks,
                 k_blocks, block_size, nnz=None, route=None):
        self.row_ptr = row_ptr
        self.col_idx = col_idx
        self.counts = counts
        self.route_batches = int(route_batches)
        self.heads = int(heads)
        self.q_blocks = int(q_blocks)
        self.k_blocks = int(k_blocks)
        self.block_size = int(block_size)
        self.nnz = nnz
        self._route = route

    @property
    def device(self):
        return self.row_ptr.device

    def nnz_value(self):
        """Total number of routed blocks (one 8-byte device-to-host read)."""
        return int(self.nnz.item())

    def to_route(self):
        """Dense boolean route [route_batches, heads, q_blocks, k_blocks]."""
        if self._route is not None:
            return self._route
        rows = self.route_batches * self.heads * self.q_blocks
        route = torch.zeros(rows, self.k_blocks, dtype=torch.bool, device=self.device)
        counts = self.counts.reshape(-1).long()
        row_ids = torch.repeat_interleave(torch.arange(rows, device=self.device), counts)
        route[row_ids, self.col_idx.long()] = True
        return route.reshape(self.route_batches, self.heads, self.q_blocks, self.k_blocks)


def csr_from_route(route, block_size=128):
    """RouteCSR of a boolean route [H,Q,K] or [R,H,Q,K] on the device.

    Column indices are the ascending selected key blocks of each row, i.e. the
    selected prefix of the reference's stable packing
    (attention_backends/layout_ops.py:128-151); built by the HIP CSR kernels.
    """
    return route_to_csr(route, block_size=block_size)


def bsa_fwd(q, k, v, csr=None, scale=None, out=None, return_lse=False, block_size=128,
            causal=False, deterministic=False, dropout_p=0.0, seed=None, offset=0):
    """Block-sparse (or, with ``csr=None``, dense) attention forward on the GPU.

    ``block_size`` (1..128) is the number of consecutive tokens per query
    block and per key block that the route addresses: 128 for ``flex_reuse``,
    the spatial tile size for the matrix-sparse backend.

    q: [B,Tq,H,D], k/v: [B,Tk,H,D], D a multiple of 8 up to 256, all bf16,
    all fp16 or all fp32 (the compute type; fp32 as split fp16 products where
    these lose nothing, else, as D above 128 for every type, on the fp32
    matrix-core kernel), on a HIP device, any strides with a contiguous head
    dim.
    ``causal`` (dense calls only): query t attends keys k <= t, as SDPA's
    is_causal.  ``deterministic`` (or
    ``torch.use_deterministic_algorithms(True)``): results reproducible bit
    for bit; otherwise a routed call may start each row's key walk where the
    other rows of its head are reading (better L2 reuse), which changes the
    fp32 accumulation order and so the last bits from run to run.
    ``dropout_p`` in (0, 1) (dense calls only): dropout on the attention
    probabilities, as SDPA's ``dropout_p``, computed in fp32 with a
    Philox4x32-10 mask drawn from ``seed`` (default: a seed from torch's CPU
    generator) and ``offset`` (dsa_bsa_fwd_dropout).  Returns O [B,Tq,H,D]
    in the input type (contiguous unless ``out`` is given) and, with
    ``return_lse``, the natural-log LSE [B,H,Tq] fp32 (of the undropped
    softmax).
    """
    lib = _lib.load()
    q = _kernel_view("q", q, attention=True)
    k = _kernel_view("k", k, q.dtype, attention=True)
    v = _kernel_view("v", v, q.dtype, attention=True)
    batch, q_tokens, heads, head_dim = q.shape
    if k.shape[0] != batch or v.shape[0] != batch or k.shape[2] != heads or v.shape[2] != heads:
        raise ValueError("q, k and v must agree on batch and heads")
    if k.shape[1] != v.shape[1]:
        raise ValueError("k and v must have the same number of tokens")
    if k.shape[3] != head_dim or v.shape[3] != head_dim:
        raise ValueError("q, k and v must share the head dimension")
    if q.device != k.device or q.device != v.device:
        raise ValueError("q, k and v must be on the same device")
    kv_tokens = k.shape[1]
    if scale is None:
        scale = head_dim ** -0.5
    if out is None:
        out = torch.empty((batch, q_tokens, heads, head_dim), dtype=q.dtype, device=q.device)
    else:
        _require_cuda("out", out)
        if out.shape != (batch, q_tokens, heads, head_dim) or out.dtype != q.dtype:
            raise ValueError("out has the wrong shape or dtype")
    lse = None
    if return_lse:
        lse = torch.empty((batch, heads, q_tokens), dtype=torch.float32, device=q.device)
    row_ptr = col_idx = None
    route_batches = 1
    if csr is not None:
        if csr.block_size != block_size:
            raise ValueError("route block size does not match block_size")
        q_blocks = math.ceil(q_tokens / block_size)
        if (csr.heads, csr.q_blocks, csr.k_blocks) != (
                heads, q_blocks, math.ceil(kv_tokens / block_size)):
            raise ValueError("route shape does not match the attention shape")
        if csr.route_batches not in (1, batch):
            raise ValueError("route batches must be 1 or the attention batch")
        if csr.row_ptr.device != q.device or csr.col_idx.device != q.device:
            raise ValueError("route must live on the attention device")
        row_ptr, col_idx = csr.row_ptr, csr.col_idx
        route_batches = csr.route_batches
    strides = _lib.int64_array(
        list(q.stride()[:3]) + list(k.stride()[:3]) + list(v.stride()[:3])
        + list(out.stride()[:3]))
    if dropout_p:
        if csr is not None:
            raise ValueError("dropout takes dense attention only")
        if not 0.0 < dropout_p < 1.0:
            raise ValueError(f"dropout_p must be in (0, 1), got {dropout_p}")
        if seed is None:
            seed = int(torch.randint(0, 2 ** 63 - 1, (), dtype=torch.int64).item())
        with torch.cuda.device(q.device):
            status = lib.dsa_bsa_fwd_dropout(
                q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                dtype_code(q.dtype, attention=True), strides, batch, q_tokens, kv_tokens,
                heads, head_dim, float(scale), int(bool(causal)), float(dropout_p),
                int(seed) & (2 ** 64 - 1), int(offset) & (2 ** 32 - 1),
                lse.data_ptr() if lse is not None else None, _stream_handle(q.device))
        _lib.check(status, "dsa_bsa_fwd_dropout")
        return (out, lse) if return_lse else out
    if not 1 <= block_size <= 128:
        raise ValueError(f"block_size {block_size} unsupported (1..128)")
    deterministic = bool(deterministic) or torch.are_deterministic_algorithms_enabled()
    # Room for the split partials of the last round of workgroups (none when
    # the key range is too short to split), or, in fp32, for the split K and V
    # (head dims above 128 run the fp32-compute kernel, which uses none); the
    # caching allocator recycles it.
    fp32_kernel = q.dtype == torch.float32 or head_dim > HEAD_DIM
    if fp32_kernel:
        workspace_bytes = _f32_workspace_bytes(lib, q, batch, heads, kv_tokens, head_dim,
                                               block_size, csr is None and not causal)
    else:
        workspace_bytes = lib.dsa_bsa_workspace_bytes_block(
            batch, heads, kv_tokens, head_dim, block_size)
    try:
        workspace = (torch.empty(workspace_bytes, dtype=torch.uint8, device=q.device)
                     if workspace_bytes else None)
    except torch.OutOfMemoryError:
        if not fp32_kernel:
            raise
        workspace, workspace_bytes = None, 0  # float32 products
    with torch.cuda.device(q.device):
        status = lib.dsa_bsa_fwd(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
            dtype_code(q.dtype, attention=True), strides,
            batch, q_tokens, kv_tokens, heads, head_dim, block_size,
            row_ptr.data_ptr() if row_ptr is not None else None,
            col_idx.data_ptr() if col_idx is not None else None,
            route_batches, float(scale), int(bool(causal)), int(bool(deterministic)),
            lse.data_ptr() if lse is not None else None,
            workspace.data_ptr() if workspace is not None else None, workspace_bytes,
            _stream_handle(q.device))
    _lib.check(status, "dsa_bsa_fwd")
    return (out, lse) if return_lse else out


def _require_bool_route(route):
    _require_cuda("route", route)
    if route.dtype != torch.bool:
        raise ValueError("route must be a boolean tensor")
    return route.contiguous()


@functools.lru_cache(maxsize=64)
def _sampled_mass_workspace_bytes(tokens, heads, block_size, samples):
    # A function of these sizes alone; a short call's time is the host's.
    return _lib.load().dsa_sampled_mass_workspace_bytes(tokens, heads, block_size, samples)


def sampled_block_mass(q, k, block_size, samples=2, scale=None):
    """Sampled block mass [heads, blocks, blocks] fp32 of a batch-1 call.

    Same contract as the reference's ``_sampled_block_mass``
    (attention_backends/flex.py:205-251), computed by one fused HIP kernel.
    """
    lib = _lib.load()
    if q.shape[0] != 1 or q.shape[1] != k.shape[1]:
        raise ValueError("sampled route update supports batch-1 self-attention")
    if samples <= 0 or samples > block_size:
        raise ValueError("route_samples must be in [1, block_size]")
    q = _kernel_view("q", q)
    k = _kernel_view("k", k, q.dtype)
    _, tokens, heads, head_dim = q.shape
    if scale is None:
        scale = head_dim ** -0.5
    blocks = math.ceil(tokens / block_size)
    mass = torch.empty((heads, blocks, blocks), dtype=torch.float32, device=q.device)
    strides = _lib.int64_array([q.stride(1), q.stride(2), k.stride(1), k.stride(2)])
    # Row sums of a single scan (none above 32 samples, which scan twice): with
    # half in several launches, without any in two scans.
    workspace_bytes = _sampled_mass_workspace_bytes(tokens, heads, block_size, samples)
    try:
        workspace = (torch.empty(workspace_bytes, dtype=torch.uint8, device=q.device)
                     if workspace_bytes else None)
    except torch.OutOfMemoryError:
        workspace = _smaller_workspace(q.device, workspace_bytes // 2, 0)
        workspace_bytes = workspace.numel() if workspace is not None else 0
    with torch.cuda.device(q.device):
        status = lib.dsa_sampled_mass_ws(
            q.data_ptr(), k.data_ptr(), dtype_code(q.dtype), strides, tokens, heads, head_dim, block_size,
            samples, float(scale), mass.data_ptr(),
            workspace.data_ptr() if workspace is not None else None, workspace_bytes,
            _stream_handle(q.device))
    _lib.check(status, "dsa_sampled_mass")
    return mass


def block_mass(q, k, lse, block_size=128, scale=None):
    """Exact block attention mass [heads, blocks, blocks] fp32 of a batch-1 call.

    Same contract as the reference's ``_block_attention_mass``
    (attention_backends/flex.py:158-202): ``lse`` is the natural-log
    normaliser of every query row ([1, H, T] or [H, T], as ``bsa_fwd(...,
    return_lse=True)`` returns it) and mass[h, qb, kb] sums
    exp(scale * q.k - lse) over the tokens of the two blocks.
    """
    lib = _lib.load()
    if q.shape[0] != 1 or q.shape[1] != k.shape[1]:
        raise ValueError("Flex bootstrap supports batch-1 self-attention")
    if block_size != 128:
        raise ValueError("The exact mass kernel currently requires block_size=128")
    q = _kernel_view("q", q)
    k = _kernel_view("k", k, q.dtype)
    _, tokens, heads, head_dim = q.shape
    _require_cuda("lse", lse)
    if lse.dtype != torch.float32:
        raise ValueError("lse must be float32")
    if lse.ndim == 3:
        if lse.shape[0] != 1:
            raise ValueError("lse must have shape [1, heads, tokens] or [heads, tokens]")
        lse = lse[0]
    if tuple(lse.shape) != (heads, tokens):
        raise ValueError("lse must have shape [1, heads, tokens] or [heads, tokens]")
    if lse.stride(1) != 1:
        lse = lse.contiguous()
    if scale is None:
        scale = head_dim ** -0.5
    blocks = math.ceil(tokens / block_size)
    mass = torch.empty((heads, blocks, blocks), dtype=torch.float32, device=q.device)
    strides = _lib.int64_array([q.stride(1), q.stride(2), k.stride(1), k.stride(2)])
    with torch.cuda.device(q.device):
        status = lib.dsa_block_mass(
            q.data_ptr(), k.data_ptr(), dtype_code(q.dtype), strides, tokens, heads, head_dim, block_size,
            lse.data_ptr(), lse.stride(0), float(scale), mass.data_ptr(),
            _stream_handle(q.device))
    _lib.check(status, "dsa_block_mass")
    return mass


def bsa_fwd_block_mass(q, k, v, scale=None):
    """Dense attention of batch-1 self-attention q/k/v [1, T, H, D] with its
    exact 128-token block mass: returns ``(out, lse, mass)`` with ``out`` and
    ``lse`` [1, H, T] as :func:`bsa_fwd` returns them and ``mass`` as
    :func:`block_mass` does (the reference's ``_dense_bootstrap`` pair of
    dense attention and ``_block_attention_mass``, attention_backends/
    flex.py:254-272, 158-202).  The mass comes from the attention launch's own
    probabilities; only head dims above 128 with T not a multiple of 128 run
    the attention and then the block-mass pass.  float32 inputs need T a
    multiple of 128.
    """
    lib = _lib.load()
    q = _kernel_view("q", q, attention=True)
    k = _kernel_view("k", k, q.dtype, attention=True)
    v = _kernel_view("v", v, q.dtype, attention=True)
    batch, tokens, heads, head_dim = q.shape
    if batch != 1 or k.shape != q.shape or v.shape != q.shape:
        raise ValueError("Flex bootstrap supports batch-1 self-attention")
    if q.device != k.device or q.device != v.device:
        raise ValueError("q, k and v must be on the same device")
    if scale is None:
        scale = head_dim ** -0.5
    blocks = math.ceil(tokens / 128)
    out = torch.empty((1, tokens, heads, head_dim), dtype=q.dtype, device=q.device)
    lse = torch.empty((1, heads, tokens), dtype=torch.float32, device=q.device)
    mass = torch.empty((heads, blocks, blocks), dtype=torch.float32, device=q.device)
    strides = _lib.int64_array(
        list(q.stride()[:3]) + list(k.stride()[:3]) + list(v.stride()[:3])
        + list(out.stride()[:3]))
    workspace_bytes = own = lib.dsa_bsa_fwd_block_mass_workspace_bytes(heads, tokens, head_dim)
    if q.dtype == torch.float32:
        workspace_bytes = _statistics_workspace_bytes(lib, q, own, heads, tokens, head_dim, 128,
                                                      True)
    try:
        workspace = torch.empty(workspace_bytes, dtype=torch.uint8, device=q.device)
    except torch.OutOfMemoryError:
        # float32 products; a partial last block: the attention, then a second pass.
        workspace = _smaller_workspace(
            q.device,
            own if tokens % 128 == 0 else lib.dsa_bsa_workspace_bytes(1, heads, tokens, head_dim))
        workspace_bytes = workspace.numel()
    with torch.cuda.device(q.device):
        status = lib.dsa_bsa_fwd_block_mass(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
            dtype_code(q.dtype, attention=True),
            strides, tokens, heads, head_dim, float(scale), lse.data_ptr(), mass.data_ptr(),
            workspace.data_ptr(), workspace_bytes, _stream_handle(q.device))
    _lib.check(status, "dsa_bsa_fwd_block_mass")
    return out, lse, mass


def tile_stats(q, k, lse, tile_shape, csr=None, scale=None, centroids=True):
    """Spatial-tile attention statistics of tile-major q/k [1, T, H, 128].

    Same quantities as the reference's matrix-sparse statistics
    (attention_backends/sparse.py:184-233 with ``csr=None``, 718-750 with the
    CSR of the attended tiles): ``lse`` is the natural-log normaliser of that
    attention ([1, H, T] or [H, T]).  Returns a dict of [H, tiles, tiles]
    tensors: ``mass`` (fp32, mass / tokens), ``mass_f16`` and, with
    ``centroids``, ``centroid_q_y``, ``centroid_q_x``, ``centroid_k_y``,
    ``centroid_k_x`` (fp16).
    """
    lib = _lib.load()
    if q.shape[0] != 1 or q.shape[1] != k.shape[1]:
        raise ValueError("tile statistics support batch-1 self-attention")
    q = _kernel_view("q", q)
    k = _kernel_view("k", k, q.dtype)
    _, tokens, heads, head_dim = q.shape
    tile_h, tile_w = (int(x) for x in tile_shape)
    tile = tile_h * tile_w
    if tile <= 0 or tokens % tile:
        raise ValueError("the tile shape must divide the token count")
    tiles = tokens // tile
    _require_cuda("lse", lse)
    if lse.dtype != torch.float32:
        raise ValueError("lse must be float32")
    if lse.ndim == 3:
        lse = lse[0]
    if tuple(lse.shape) != (heads, tokens):
        raise ValueError("lse must have shape [1, heads, tokens] or [heads, tokens]")
    if lse.stride(1) != 1:
        lse = lse.contiguous()
    if scale is None:
        scale = head_dim ** -0.5
    row_ptr = col_idx = None
    if csr is not None:
        if (csr.route_batches, csr.heads, csr.q_blocks, csr.k_blocks) != (1, heads, tiles, tiles):
            raise ValueError("route shape does not match the tile layout")
        row_ptr, col_idx = csr.row_ptr, csr.col_idx
    shape = (heads, tiles, tiles)
    out = {"mass": torch.empty(shape, dtype=torch.float32, device=q.device),
           "mass_f16": torch.empty(shape, dtype=torch.float16, device=q.device)}
    names = ("centroid_q_y", "centroid_q_x", "centroid_k_y", "centroid_k_x")
    if centroids:
        for name in names:
            out[name] = torch.empty(shape, dtype=torch.float16, device=q.device)
    strides = _lib.int64_array([q.stride(1), q.stride(2), k.stride(1), k.stride(2)])
    with torch.cuda.device(q.device):
        status = lib.dsa_tile_stats(
            q.data_ptr(), k.data_ptr(), dtype_code(q.dtype), strides, tokens, heads, head_dim, tile_h, tile_w,
            lse.data_ptr(), lse.stride(0),
            row_ptr.data_ptr() if row_ptr is not None else None,
            col_idx.data_ptr() if col_idx is not None else None, float(scale),
            out["mass"].data_ptr(), out["mass_f16"].data_ptr(),
            *[out[name].data_ptr() if name in out else None for name in names],
            _stream_handle(q.device))
    _lib.check(status, "dsa_tile_stats")
    return out


def bsa_fwd_tile_stats(q, k, v, csr, tile_shape, scale=None, deterministic=False,
                       centroids=True):
    """One matrix-sparse step: attention of tile-major q/k/v [1, T, H, D] over
    the CSR of kept tiles (``csr=None``: every tile, dense) and the statistics
    of that same softmax (the reference's ``sparse_chunk``, attention_backends/
    sparse.py:670-751; dense: ``_dense_route``, 184-233).  Returns
    ``(out, lse, stats)`` with ``out`` as :func:`bsa_fwd` returns it, ``lse``
    [1, H, T] and ``stats`` as :func:`tile_stats` returns them.  Every call
    gets its statistics from the attention launch itself (per query row and
    key tile), which a short second launch combines per cell; no second QK
    pass runs.  ``deterministic`` as in :func:`bsa_fwd`: without it (and
    without torch's deterministic mode) a routed call's output, mass and
    centroids can differ in the last bits from run to run.
    """
    lib = _lib.load()
    q = _kernel_view("q", q, attention=True)
    k = _kernel_view("k", k, q.dtype, attention=True)
    v = _kernel_view("v", v, q.dtype, attention=True)
    batch, tokens, heads, head_dim = q.shape
    if batch != 1 or k.shape != q.shape or v.shape != q.shape:
        raise ValueError("tile statistics support batch-1 self-attention")
    if q.device != k.device or q.device != v.device:
        raise ValueError("q, k and v must be on the same device")
    tile_h, tile_w = (int(x) for x in tile_shape)
    tile = tile_h * tile_w
    if tile <= 0 or tile > 128 or tokens % tile:
        raise ValueError("the tile shape must divide the token count (1..128 tokens per tile)")
    tiles = tokens // tile
    if csr is not None:
        if (csr.route_batches, csr.heads, csr.q_blocks, csr.k_blocks, csr.block_size) != (
                1, heads, tiles, tiles, tile):
            raise ValueError("route shape does not match the tile layout")
        if csr.row_ptr.device != q.device or csr.col_idx.device != q.device:
            raise ValueError("route must live on the attention device")
        # Room for every entry the list can hold where that is little (a caller's
        # own list may name a tile twice); else for the listed ones, whose number
        # the device holds (a read that waits for it).
        entries = csr.col_idx.numel()
        if entries * tile > MAX_UNCOUNTED_ROWS:
            entries = csr.nnz_value() if csr.nnz is not None else int(csr.row_ptr[-1].item())
    else:
        entries = heads * tiles * tiles
    if scale is None:
        scale = head_dim ** -0.5
    deterministic = bool(deterministic) or torch.are_deterministic_algorithms_enabled()
    out = torch.empty((1, tokens, heads, head_dim), dtype=q.dtype, device=q.device)
    lse = torch.empty((1, heads, tokens), dtype=torch.float32, device=q.device)
    shape = (heads, tiles, tiles)
    stats = {"mass": torch.empty(shape, dtype=torch.float32, device=q.device),
             "mass_f16": torch.empty(shape, dtype=torch.float16, device=q.device)}
    names = ("centroid_q_y", "centroid_q_x", "centroid_k_y", "centroid_k_x")
    if centroids:
        for name in names:
            stats[name] = torch.empty(shape, dtype=torch.float16, device=q.device)
    strides = _lib.int64_array(
        list(q.stride()[:3]) + list(k.stride()[:3]) + list(v.stride()[:3])
        + list(out.stride()[:3]))
    workspace_bytes = own = lib.dsa_bsa_fwd_tile_stats_workspace_bytes(
        heads, tokens, head_dim, tile_h, tile_w, entries)
    if q.dtype == torch.float32:
        workspace_bytes = _statistics_workspace_bytes(lib, q, own, heads, tokens, head_dim, tile,
                                                      csr is None)
    try:
        workspace = (torch.empty(workspace_bytes, dtype=torch.uint8, device=q.device)
                     if workspace_bytes else None)
    except torch.OutOfMemoryError:
        if workspace_bytes == own:
            raise
        workspace, workspace_bytes = _smaller_workspace(q.device, own), own  # float32 products
    with torch.cuda.device(q.device):
        status = lib.dsa_bsa_fwd_tile_stats(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
            dtype_code(q.dtype, attention=True), strides, tokens, heads, head_dim, tile_h, tile_w,
            csr.row_ptr.data_ptr() if csr is not None else None,
            csr.col_idx.data_ptr() if csr is not None else None,
            entries, float(scale), int(bool(deterministic)),
            lse.data_ptr(), stats["mass"].data_ptr(), stats["mass_f16"].data_ptr(),
            *[stats[name].data_ptr() if name in stats else None for name in names],
            workspace.data_ptr() if workspace is not None else None, workspace_bytes,
            _stream_handle(q.device))
    _lib.check(status, "dsa_bsa_fwd_tile_stats")
    return out, lse, stats


def route_select(mass, target, keep, previous=None, persistence=0.0, sink_blocks=0):
    """Prior + top-mass selection + sink on the GPU.

    mass: fp32 [..., K] (non-negative); previous: bool of the same shape or
    None.  Returns (route bool [..., K], counts int32 [...]).  The cap is
    max(1, ceil(K * keep)) exactly as the reference's ``_top_mass_route``
    (attention_backends/flex.py:83-94).
    """
    lib = _lib.load()
    _require_cuda("mass", mass)
    if mass.dtype != torch.float32:
        raise ValueError("mass must be float32")
    if not 0 < keep <= 1:
        raise ValueError("keep must be in (0, 1]")
    if not 0 < target <= 1:
        raise ValueError("mass_target must be in (0, 1]")
    mass = mass.contiguous()
    keys = mass.shape[-1]
    rows = mass.numel() // keys
    cap = max(1, math.ceil(keys * keep))
    prev_ptr = None
    if previous is not None and persistence:
        previous = _require_bool_route(previous)
        if previous.shape != mass.shape:
            raise ValueError("previous route must match the mass shape")
        prev_ptr = previous.data_ptr()
    route = torch.empty(mass.shape, dtype=torch.bool, device=mass.device)
    counts = torch.empty(mass.shape[:-1], dtype=torch.int32, device=mass.device)
    with torch.cuda.device(mass.device):
        status = lib.dsa_route_select(
            mass.data_ptr(), prev_ptr, rows, keys, float(persistence), float(target), cap,
            int(sink_blocks), route.data_ptr(), counts.data_ptr(), _stream_handle(mass.device))
    _lib.check(status, "dsa_route_select")
    return route, counts


def _neighbor_table(neighbors, blocks, device):
    _require_cuda("neighbors", neighbors)
    if tuple(neighbors.shape) != (blocks, 4):
        raise ValueError("neighbors must have shape [blocks, 4]")
    if neighbors.device != device:
        raise ValueError("neighbors must live on the route device")
    return neighbors.to(torch.int32).contiguous()


def frontier_mask(route, neighbors, return_count=False):
    """Selected route cells with an unselected valid neighbour along the query
    or key axis (attention_backends/routing.py:35-41).  route: bool [H, B, B];
    neighbors: int [B, 4] (-1 = none).  With ``return_count`` also returns the
    number of frontier cells as a device int64 tensor."""
    lib = _lib.load()
    route = _require_bool_route(route)
    if route.ndim != 3 or route.shape[1] != route.shape[2]:
        raise ValueError("route must have shape [heads, blocks, blocks]")
    heads, blocks, _ = route.shape
    neighbors = _neighbor_table(neighbors, blocks, route.device)
    frontier = torch.empty_like(route)
    count = torch.empty(1, dtype=torch.int64, device=route.device) if return_count else None
    with torch.cuda.device(route.device):
        status = lib.dsa_frontier_mask(
            route.data_ptr(), heads, blocks, neighbors.data_ptr(), frontier.data_ptr(),
            count.data_ptr() if count is not None else None, _stream_handle(route.device))
    _lib.check(status, "dsa_frontier_mask")
    return (frontier, count) if return_count else frontier


def directional_update(mass, previous, neighbors, *, keep, persistence=0.5, min_ratio=0.0,
                       candidate_bonus=0.0, budget_scale=1.0, exploration_fraction=0.0,
                       expand_q=True, expand_k=True, expand_joint=True,
                       previous_frontier=None, sink_blocks=0):
    """Frontier-aware directional route update on the GPU.

    Same contract as the reference's ``directional_budget_update``
    (attention_backends/routing.py:92-168), followed by the first
    ``sink_blocks`` columns (flex.py:544-546).  Returns a dict with route
    (after the sink), counts (int32 [H, B], sink included), candidates,
    exploration, dropped and added (the last two before the sink, as the
    reference reports them).
    """
    lib = _lib.load()
    _require_cuda("mass", mass)
    if mass.dtype != torch.float32:
        raise ValueError("mass must be float32")
    previous = _require_bool_route(previous)
    if previous.shape != mass.shape:
        raise ValueError("previous route and mass must have identical shapes")
    if mass.ndim != 3 or mass.shape[1] != mass.shape[2]:
        raise ValueError("mass must have shape [heads, blocks, blocks]")
    if budget_scale <= 0:
        raise ValueError("budget_scale must be positive")
    if not 0 <= exploration_fraction <= 1:
        raise ValueError("exploration_fraction must be in [0, 1]")
    heads, blocks, _ = mass.shape
    mass = mass.contiguous()
    neighbors = _neighbor_table(neighbors, blocks, mass.device)
    if previous_frontier is not None:
        previous_frontier = _require_bool_route(previous_frontier)
        if previous_frontier.shape != mass.shape:
            raise ValueError("previous_frontier must match the route shape")
    cap = max(1, math.ceil(blocks * keep))
    explore = max(1, math.ceil(blocks * exploration_fraction)) if exploration_fraction else 0
    flags = (1 if expand_q else 0) | (2 if expand_k else 0) | (4 if expand_joint else 0)
    outputs = {name: torch.empty(mass.shape, dtype=torch.bool, device=mass.device)
               for name in ("route", "candidates", "exploration", "dropped", "added")}
    counts = torch.empty((heads, blocks), dtype=torch.int32, device=mass.device)
    with torch.cuda.device(mass.device):
        status = lib.dsa_directional_update(
            mass.data_ptr(), previous.data_ptr(),
            previous_frontier.data_ptr() if previous_frontier is not None else None,
            neighbors.data_ptr(), heads, blocks, cap, float(persistence), float(min_ratio),
            float(candidate_bonus), float(budget_scale), explore, flags, int(sink_blocks),
            outputs["route"].data_ptr(), counts.data_ptr(), outputs["candidates"].data_ptr(),
            outputs["exploration"].data_ptr(), outputs["dropped"].data_ptr(),
            outputs["added"].data_ptr(), _stream_handle(mass.device))
    _lib.check(status, "dsa_directional_update")
    outputs["counts"] = counts
    return outputs


def drop_low_mass(mask, mass, drop_factor, sink_tiles=0):
    """Next route of the matrix-sparse backend (attention_backends/sparse.py:
    327-348, then the first ``sink_tiles`` columns): returns (route bool, counts
    int32).  ``mass`` is fp16 (the stored route mass) or fp32."""
    lib = _lib.load()
    mask = _require_bool_route(mask)
    _require_cuda("mass", mass)
    if mask.ndim != 3 or mask.shape[1] != mask.shape[2] or mass.shape != mask.shape:
        raise ValueError("mask and mass must have shape [heads, tiles, tiles]")
    if mass.dtype not in (torch.float16, torch.float32):
        raise ValueError("mass must be float16 or float32")
    heads, tiles, _ = mask.shape
    mass = mass.contiguous()
    out = torch.empty_like(mask)
    counts = torch.empty((heads, tiles), dtype=torch.int32, device=mask.device)
    scratch = torch.empty(4 * heads, dtype=torch.float32, device=mask.device)
    with torch.cuda.device(mask.device):
        status = lib.dsa_drop_low_mass(
            mask.data_ptr(), mass.data_ptr(), int(mass.dtype == torch.float16), heads, tiles,
            float(drop_factor), int(sink_tiles), scratch.data_ptr(), out.data_ptr(),
            counts.data_ptr(), _stream_handle(mask.device))
    _lib.check(status, "dsa_drop_low_mass")
    return out, counts


EXPAND_POLICIES = {"all": 1, "directional": 2}


def expand_route(mask, grid_tiles, policy, mass=None, centroids=None, centroid_threshold=0.15,
                 huge_factor=2.0):
    """Predicted next mask (attention_backends/sparse.py:350-373) for policy
    "all" or "directional".  ``grid_tiles`` = (frames, blocks_h, blocks_w);
    ``mass`` and ``centroids`` (q_y, q_x, k_y, k_x) are fp16 [H, tiles, tiles]."""
    lib = _lib.load()
    if policy not in EXPAND_POLICIES:
        raise ValueError(f"unknown expansion policy {policy!r}")
    mask = _require_bool_route(mask)
    heads, tiles, _ = mask.shape
    frames, blocks_h, blocks_w = (int(x) for x in grid_tiles)
    if frames * blocks_h * blocks_w != tiles:
        raise ValueError("the tile grid does not match the route")
    pointers = [None] * 5
    scratch = None
    if policy == "directional":
        tensors = [mass, *centroids]
        for tensor in tensors:
            _require_cuda("mass/centroid", tensor)
            if tensor.dtype != torch.float16 or tensor.shape != mask.shape:
                raise ValueError("directional expansion needs fp16 mass and centroids")
        tensors = [tensor.contiguous() for tensor in tensors]
        pointers = [tensor.data_ptr() for tensor in tensors]
        scratch = torch.empty(4 * heads, dtype=torch.float32, device=mask.device)
    out = torch.empty_like(mask)
    with torch.cuda.device(mask.device):
        status = lib.dsa_expand_route(
            mask.data_ptr(), *pointers, heads, frames, blocks_h, blocks_w,
            EXPAND_POLICIES[policy], float(centroid_threshold), float(huge_factor),
            scratch.data_ptr() if scratch is not None else None, out.data_ptr(),
            _stream_handle(mask.device))
    _lib.check(status, "dsa_expand_route")
    return out


def route_to_csr(route, counts=None, block_size=128):
    """GPU CSR of a boolean route [H,Q,K] or [R,H,Q,K] (ascending key blocks)."""
    lib = _lib.load()
    route = _require_bool_route(route)
    if route.ndim == 3:
        route = route.unsqueeze(0)
    if route.ndim != 4:
        raise ValueError("route must have shape [heads, Q, K] or [batch, heads, Q, K]")
    route_batches, heads, q_blocks, k_blocks = route.shape
    rows = route_batches * heads * q_blocks
    device = route.device
    counts_out = None
    if counts is None:
        counts_out = torch.empty((route_batches, heads, q_blocks), dtype=torch.int32,
                                 device=device)
    else:
        counts = counts.reshape(route_batches, heads, q_blocks).to(torch.int32).contiguous()
    row_ptr = torch.empty(rows + 1, dtype=torch.int32, device=device)
    col_idx = torch.empty(max(1, route.numel()), dtype=torch.int32, device=device)
    nnz = torch.empty(1, dtype=torch.int64, device=device)
    with torch.cuda.device(device):
        status = lib.dsa_route_to_csr(
            route.data_ptr(), rows, k_blocks,
            counts.data_ptr() if counts is not None else None,
            counts_out.data_ptr() if counts_out is not None else None,
            row_ptr.data_ptr(), col_idx.data_ptr(), nnz.data_ptr(), _stream_handle(device))
    _lib.check(status, "dsa_route_to_csr")
    return RouteCSR(row_ptr, col_idx, counts if counts is not None else counts_out,
                    route_batches, heads, q_blocks, k_blocks, block_size, nnz=nnz,
                    route=route)


def pack_rows(route):
    """(counts int32 [...], indices int32 [..., K]): selected ids ascending,
    then unselected ids ascending (layout_ops.py:128-151 semantics)."""
    lib = _lib.load()
    route = _require_bool_route(route)
    if route.ndim < 2:
        raise ValueError("route must be a boolean tensor with at least two axes")
    keys = route.shape[-1]
    rows = route.numel() // keys
    counts = torch.empty(route.shape[:-1], dtype=torch.int32, device=route.device)
    indices = torch.empty(route.shape, dtype=torch.int32, device=route.device)
    with torch.cuda.device(route.device):
        status = lib.dsa_pack_rows(route.data_ptr(), rows, keys, counts.data_ptr(),
                                   indices.data_ptr(), _stream_handle(route.device))
    _lib.check(status, "dsa_pack_rows")
    return counts, indices


def permute_tokens(tensors, permutation, out=None, head_major=False):
    """Gather along the token axis: out[n][b, t] = tensors[n][b, permutation[t]].

    tensors: 1-3 CUDA tensors [B, T, H, D] sharing shape and dtype, any
    strides with a contiguous last axis.  permutation: int32 [T] on the device.
    Outputs are [B, T, H, D]; contiguous, or views of head-major (BHSD)
    storage with ``head_major=True``.  Bit-exact.
    """
    lib = _lib.load()
    tensors = list(tensors)
    if not 1 <= len(tensors) <= 3:
        raise ValueError("permute_tokens moves 1 to 3 tensors")
    first = tensors[0]
    for index, tensor in enumerate(tensors):
        _require_cuda(f"tensor {index}", tensor)
        if tensor.shape != first.shape or tensor.dtype != first.dtype:
            raise ValueError("tensors must share shape and dtype")
        if tensor.ndim != 4:
            raise ValueError("tensors must have shape [batch, tokens, heads, dim]")
    _require_cuda("permutation", permutation)
    if permutation.ndim != 1 or permutation.numel() != first.shape[1]:
        raise ValueError("permutation must contain one index per token")
    permutation = permutation.to(torch.int32).contiguous()
    batch, tokens, heads, dim = first.shape
    element = first.element_size()
    sources = []
    for tensor in tensors:
        ok = (tensor.stride(3) == 1
              and all((stride * element) % 16 == 0 for stride in tensor.stride()[:3])
              and tensor.data_ptr() % 16 == 0)
        sources.append(tensor if ok else tensor.contiguous())
    if out is None:
        if head_major:
            out = [torch.empty((batch, heads, tokens, dim), dtype=first.dtype,
                               device=first.device).transpose(1, 2) for _ in sources]
        else:
            out = [torch.empty_like(first, memory_format=torch.contiguous_format)
                   for _ in sources]
    if (dim * element) % 16 != 0:
        raise ValueError("rows must be a multiple of 16 bytes")
    src_strides = _lib.int64_array(
        [s * element for tensor in sources for s in tensor.stride()[:3]])
    dst_strides = _lib.int64_array(
        [s * element for tensor in out for s in tensor.stride()[:3]])
    with torch.cuda.device(first.device):
        status = lib.dsa_permute_rows(
            len(sources), _lib.pointer_array([t.data_ptr() for t in sources]),
            _lib.pointer_array([t.data_ptr() for t in out]), src_strides, dst_strides,
            permutation.data_ptr(), batch, tokens, heads, dim * element,
            _stream_handle(first.device))
    _lib.check(status, "dsa_permute_rows")
    return out


# ---------------------------------------------------------------------------
# Wan DiT block elementwise work (end-to-end loop)
# ---------------------------------------------------------------------------

def _rows_view(name, x):
    _require_cuda(name, x)
    if x.dtype != torch.bfloat16:
        raise ValueError(f"{name} must be bfloat16")
    if x.stride(-1) != 1:
        x = x.contiguous()
    dim = x.shape[-1]
    rows = x.numel() // dim
    flat = x.reshape(rows, dim) if x.is_contiguous() else x.contiguous().reshape(rows, dim)
    return flat


def _f32_or_none(name, t, device):
    if t is None:
        return None
    _require_cuda(name, t)
    if t.dtype != torch.float32:
        raise ValueError(f"{name} must be float32")
    if t.device != device:
        raise ValueError(f"{name} must live on the tensor's device")
    t = t.contiguous()
    # The kernels read parameter vectors with 16-byte loads.
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _out_rows(out, x, rows, dim):
    """A [rows, dim] view of the caller's output tensor (or a new one)."""
    if out is None:
        return torch.empty((rows, dim), dtype=torch.bfloat16, device=x.device)
    if out.dtype != torch.bfloat16 or out.device != x.device or out.shape != x.shape:
        raise ValueError("out must be a bfloat16 tensor of x's shape on x's device")
    try:
        return out.view(rows, dim)
    except RuntimeError as exc:
        raise ValueError("out must be viewable as [rows, dim] rows") from exc


def _row_groups(name, t, rows, dim):
    """Rows per group of a per-group fp32 parameter [groups, dim]."""
    if t.numel() % dim or t.shape[-1] != dim:
        raise ValueError(f"{name} must be [groups, {dim}]")
    groups = t.numel() // dim
    if rows % groups:
        raise ValueError(f"{name} has {groups} groups, which do not divide {rows} rows")
    return rows // groups


def layernorm_modulate(x, shift=None, scale=None, weight=None, bias=None, eps=1e-6, out=None):
    """LN(x) [* weight + bias] [* (1 + scale) + shift] over the last axis of a
    bf16 [B, T, C] tensor; shift/scale fp32 [B, C] (one vector per batch item)."""
    lib = _lib.load()
    flat = _rows_view("x", x)
    rows, dim = flat.shape
    weight, bias, shift, scale = (_f32_or_none(n, t, x.device) for n, t in (
        ("weight", weight), ("bias", bias), ("shift", shift), ("scale", scale)))
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and t.numel() != dim:
            raise ValueError(f"{name} must hold {dim} values")
    per_group = _row_groups("scale", scale, rows, dim) if scale is not None else rows
    if shift is not None and (scale is None or shift.shape != scale.shape):
        raise ValueError("shift needs a scale of the same shape")
    rows_out = _out_rows(out, x, rows, dim)
    with torch.cuda.device(x.device):
        status = lib.dsa_layernorm_modulate(
            flat.data_ptr(), flat.stride(0), rows, dim,
            *[t.data_ptr() if t is not None else None for t in (weight, bias, shift, scale)],
            per_group, float(eps), rows_out.data_ptr(), rows_out.stride(0),
            _stream_handle(x.device))
    _lib.check(status, "dsa_layernorm_modulate")
    return out if out is not None else rows_out.view(x.shape)


def rmsnorm_rope(x, weight, head_dim=128, cos_sin=None, eps=1e-6, out=None):
    """rope(RMSNorm(x) * weight) over the last axis of bf16 [B, T, C]; cos_sin
    fp32 [T, head_dim / 2, 2] or None (no rotation)."""
    lib = _lib.load()
    flat = _rows_view("x", x)
    rows, dim = flat.shape
    weight = _f32_or_none("weight", weight, x.device)
    cos_sin = _f32_or_none("cos_sin", cos_sin, x.device)
    tokens = x.shape[-2] if x.ndim >= 2 else rows
    if weight.numel() != dim:
        raise ValueError(f"weight must hold {dim} values")
    if cos_sin is not None and cos_sin.numel() != tokens * head_dim:
        raise ValueError(f"cos_sin must be [{tokens}, {head_dim // 2}, 2]")
    rows_out = _out_rows(out, x, rows, dim)
    with torch.cuda.device(x.device):
        status = lib.dsa_rmsnorm_rope(
            flat.data_ptr(), flat.stride(0), rows, dim, head_dim, weight.data_ptr(),
            cos_sin.data_ptr() if cos_sin is not None else None, tokens, float(eps),
            rows_out.data_ptr(), rows_out.stride(0), _stream_handle(x.device))
    _lib.check(status, "dsa_rmsnorm_rope")
    return out if out is not None else rows_out.view(x.shape)


def gated_residual(x, y, gate=None, out=None):
    """x + gate * y over bf16 [B, T, C]; gate fp32 [B, C] or None (1)."""
    lib = _lib.load()
    fx = _rows_view("x", x)
    fy = _rows_view("y", y)
    if fx.shape != fy.shape:
        raise ValueError("x and y must have the same shape")
    rows, dim = fx.shape
    gate = _f32_or_none("gate", gate, x.device)
    per_group = _row_groups("gate", gate, rows, dim) if gate is not None else rows
    rows_out = _out_rows(out, x, rows, dim)
    with torch.cuda.device(x.device):
        status = lib.dsa_gated_residual(
            fx.data_ptr(), fx.stride(0), fy.data_ptr(), fy.stride(0),
            gate.data_ptr() if gate is not None else None, rows, dim, per_group,
            rows_out.data_ptr(), rows_out.stride(0), _stream_handle(x.device))
    _lib.check(status, "dsa_gated_residual")
    return out if out is not None else rows_out.view(x.shape)


# ---------------------------------------------------------------------------
# Sequences of different lengths: a paged key/value cache and the attentions
# around it
# ---------------------------------------------------------------------------

_I64x2, _I64x6, _I64x8 = ctypes.c_int64 * 2, ctypes.c_int64 * 6, ctypes.c_int64 * 8
_I64x10, _I64x14 = ctypes.c_int64 * 10, ctypes.c_int64 * 14


class PagedPlan(typing.NamedTuple):
    """Where a step's new tokens go (``paged_plan``); all on the device."""

    q_start: torch.Tensor  # int32 [requests + 1]: new tokens before each request
    kv_lens: torch.Tensor  # int32 [requests]: cached and new tokens
    slots: torch.Tensor    # int64 [tokens]: page * page_size + row, -1: no place
    status: torch.Tensor   # int32 [2]: pages needed, new tokens without a slot


# Short calls (a plan, a step's write, a decoding step of a few requests) are bound
# by the host: the helpers below look at each tensor once.  Lean forms of the
# checks and no device context where the device is current took a plan from 13.0
# to 10.9 us, and those and the checks kept per layout (below) a step's write from
# 14.3 to 7.2 us.

def _call(function, what, device, *args):
    """One libdsa call on the device's current stream (its last argument)."""
    if torch._C._cuda_getDevice() == device.index:
        status = function(*args, torch._C._cuda_getCurrentRawStream(device.index))
    else:
        with torch.cuda.device(device):
            status = function(*args, torch._C._cuda_getCurrentRawStream(device.index))
    if status != _lib.DSA_OK:
        _lib.check(status, what)


def _index_vector(name, t, device, size=None):
    _require_cuda(name, t)
    if t.dtype != torch.int32 or t.ndim != 1:
        raise ValueError(f"{name} must be a one-dimensional int32 tensor")
    if t.device != device:
        raise ValueError(f"{name} must live on {device}")
    if size is not None and t.shape[0] != size:
        raise ValueError(f"{name} must hold {size} values, got {t.shape[0]}")
    return t if t.is_contiguous() else t.contiguous()


def _block_table(t, device, requests):
    """(address, row stride, row length) of a block table."""
    _require_cuda("block_table", t)
    if t.dtype != torch.int32 or t.ndim != 2:
        raise ValueError("block_table must be an int32 tensor [requests, pages per request]")
    rows, width = t.shape
    if t.device != device or rows != requests:
        raise ValueError(f"block_table must have {requests} rows on {device}")
    if t.is_contiguous():
        return t.data_ptr(), width, width
    stride = t.stride()
    if stride[1] != 1 or (requests > 1 and stride[0] < width):
        raise ValueError("block_table rows must be contiguous and apart")
    return t.data_ptr(), max(stride[0], width), width


def _page_size(value):
    if not 16 <= value <= 1 << 30 or value & (value - 1):
        raise ValueError(f"page_size {value} unsupported (a power of two from 16)")


def _row_strides(shape, strides, size):
    """Element strides of all axes but the last of a tensor of `size`-byte elements,
    0 for axes of one entry; None where the kernels cannot address it in place: its
    last axis is not contiguous, or a row not a multiple of 16 bytes from another."""
    *lead, last = strides
    if last != 1 and shape[-1] != 1:
        return None
    mask = 16 // size - 1
    for axis, stride in enumerate(lead):
        if shape[axis] == 1:
            lead[axis] = 0
        elif stride & mask:
            return None
    return lead


def _layout(t):
    return t.shape, t.stride(), t.dtype


def _cache_strides(name, layout, dtype):
    """Strides of a [pages, page_size, kv_heads, head_dim] cache, used in place."""
    shape, strides, own = layout
    if len(shape) != 4:
        raise ValueError(f"{name} must have shape [pages, page_size, kv_heads, head_dim]")
    if own != dtype:
        raise ValueError(f"{name} must be {dtype}, got {own}")
    strides = _row_strides(shape, strides, dtype.itemsize)
    if strides is None:
        if 0 not in shape:
            raise ValueError(f"{name} must have a contiguous, 16-byte aligned head dimension")
        strides = [0, 0, 0]
    return strides


def _apart(name, layout):
    """Refuses a tensor to write into whose rows share memory (an expanded one)."""
    shape, strides, _ = layout
    if any(stride == 0 and size > 1 for stride, size in zip(strides, shape)):
        raise ValueError(f"{name} is written in place and must not be an expanded view")


def _sequence_strides(name, layout, dtype):
    """Strides of a [rows, heads, head_dim] operand, None: to be copied."""
    shape, strides, own = layout
    if len(shape) != 3:
        raise ValueError(f"{name} must have shape [rows, heads, head_dim]")
    if own != dtype:
        raise ValueError(f"{name} must be {dtype} like q, got {own}")
    if shape[0] >= 1 << 31:
        raise ValueError(f"{name} must have fewer than 2^31 rows")
    return _row_strides(shape, strides, dtype.itemsize)


def _aligned(name, t):
    if t.data_ptr() & 15 and t.numel():
        raise ValueError(f"{name} must have a contiguous, 16-byte aligned head dimension")


def _in_place(copies, *operands):
    """The operands, copied where the kernels cannot read them in place: those of
    `copies`, and those at an address that is no multiple of 16 bytes."""
    return [t.clone(memory_format=torch.contiguous_format) if i in copies or t.data_ptr() & 15
            else t for i, t in enumerate(operands)]


def paged_plan(cached, new, block_table, free_pages, page_size, tokens, free_start=None):
    """Places for a step's new tokens in a paged key/value cache.

    ``cached`` and ``new`` (int32 [requests], on the device): tokens of every
    request in the cache, and new ones.  Request r's pages are listed in
    ``block_table[r]`` (int32); the first ceil(cached / page_size) entries are
    its own already, and the pages its new tokens need beyond them are taken
    from ``free_pages`` (int32, in request order) and entered in its row, in
    place.  ``tokens`` is the length of the slot map: at least the sum of
    ``new``, which the host need not know exactly.  Nothing is read back; at
    most 8,192 requests.

    ``free_start`` (int32 [1] on the device): pages of ``free_pages`` given out
    before; the plan takes those behind them.  The call leaves it as it is, so
    that a repeated call gives the same plan; ``free_start += plan.status[:1]``
    takes the pages off the list.  A step that is captured and replayed needs it
    (and that addition in the capture): without it every replay starts at the
    list's first page again, and gives pages out twice.

    Returns a ``PagedPlan``: ``q_start``, ``kv_lens`` for ``paged_attention``,
    ``slots`` for ``paged_write`` (-1 behind the last request's tokens, and for
    tokens without a page: ``free_pages`` or the table's row is too short, or the
    page's entry in either is negative), and ``status`` = (pages needed, new tokens
    without a slot, those behind ``tokens`` among them): the caller's free list
    starts behind the first ``status[0]`` pages next time.  A step that lost tokens
    (``status[1]``) is not continued, for ``kv_lens`` counts tokens that are
    nowhere: the same call, from the same ``cached`` and ``free_start``, is made
    again once there are pages, and the step's keys are written again.
    """
    lib = _lib.load()
    _require_cuda("cached", cached)
    device = cached.device
    cached = _index_vector("cached", cached, device)
    requests = cached.shape[0]
    new = _index_vector("new", new, device, requests)
    table, table_stride, width = _block_table(block_table, device, requests)
    free_pages = _index_vector("free_pages", free_pages, device)
    if free_start is not None:
        free_start = _index_vector("free_start", free_start, device, 1)
    _page_size(page_size)
    if not 0 <= tokens < 1 << 31:
        raise ValueError(f"tokens must be in [0, 2^31), got {tokens}")
    ints = torch.empty(2 * requests + 3, dtype=torch.int32, device=device)
    slots = torch.empty(tokens, dtype=torch.int64, device=device)
    base = ints.data_ptr()
    _call(lib.dsa_paged_plan_from, "dsa_paged_plan", device, cached.data_ptr(), new.data_ptr(),
          requests, table, table_stride, width, free_pages.data_ptr(), free_pages.shape[0],
          None if free_start is None else free_start.data_ptr(), page_size, tokens, base,
          base + 4 * (requests + 1), slots.data_ptr(), base + 4 * (2 * requests + 1))
    q_start, kv_lens, status = torch.split_with_sizes(ints, (requests + 1, requests, 2))
    return PagedPlan(q_start, kv_lens, slots, status)


# What a call's shapes, strides and types decide is checked once per combination of
# them (a step's write 11.4 -> 7.2 us); addresses and devices are looked at each time.
@functools.lru_cache(maxsize=512)
def _write_layout(k, v, k_cache, v_cache):
    """(operands to copy first, strides in bytes, tokens, heads, row bytes, pages, page size)."""
    dtype = k[2]
    if dtype.itemsize not in (2, 4):
        raise ValueError(f"paged_write moves elements of 2 or 4 bytes, not {dtype}")
    rows = [_sequence_strides("k", k, dtype), _sequence_strides("v", v, dtype)]
    caches = [_cache_strides("k_cache", k_cache, dtype), _cache_strides("v_cache", v_cache, dtype)]
    tokens, heads, head_dim = k[0]
    pages, page_size, cache_heads, cache_dim = k_cache[0]
    if v[0] != k[0] or v_cache[0] != k_cache[0]:
        raise ValueError("k and v, and their caches, must have the same shape")
    if cache_heads != heads or cache_dim != head_dim:
        raise ValueError("the caches and k must agree on heads and head dimension")
    _page_size(page_size)
    if head_dim * dtype.itemsize % 16:
        raise ValueError("rows must be a multiple of 16 bytes")
    _apart("k_cache", k_cache)
    _apart("v_cache", v_cache)
    copies = tuple(i for i, x in enumerate(rows) if x is None)
    strides = None if copies else _I64x10(*[x * dtype.itemsize for t in rows + caches for x in t])
    return copies, strides, tokens, heads, head_dim * dtype.itemsize, pages, page_size


def paged_write(k, v, k_cache, v_cache, slots):
    """Writes keys and values [tokens, kv_heads, head_dim] into the caches
    [pages, page_size, kv_heads, head_dim], row t at slot ``slots[t]`` (int64 on
    the device; page * page_size + row).  Rows whose slot lies outside the cache
    (-1) are skipped.  A call's slots are distinct, as ``paged_plan`` gives
    them: of rows that share one, parts of either may be kept.  k and v do not
    overlap the caches.  Any element type of 2 or 4 bytes."""
    lib = _lib.load()
    for name, t in (("k", k), ("v", v), ("k_cache", k_cache), ("v_cache", v_cache),
                    ("slots", slots)):
        _require_cuda(name, t)
    copies, strides, tokens, heads, row_bytes, pages, page_size = _write_layout(
        _layout(k), _layout(v), _layout(k_cache), _layout(v_cache))
    if slots.dtype != torch.int64 or slots.shape != (tokens,):
        raise ValueError(f"slots must be an int64 tensor of {tokens} values")
    device = k_cache.device
    if not (k.device == v.device == v_cache.device == slots.device == device):
        raise ValueError("k, v, the caches and slots must be on the same device")
    _aligned("k_cache", k_cache)
    _aligned("v_cache", v_cache)
    if tokens == 0 or pages == 0 or heads == 0 or row_bytes == 0:
        return
    if copies or (k.data_ptr() | v.data_ptr()) & 15:
        return paged_write(*_in_place(copies, k, v), k_cache, v_cache, slots)
    if not slots.is_contiguous():
        slots = slots.contiguous()
    _call(lib.dsa_paged_write, "dsa_paged_write", device, k.data_ptr(), v.data_ptr(),
          k_cache.data_ptr(), v_cache.data_ptr(), strides, tokens, heads, row_bytes, pages,
          page_size, slots.data_ptr())


@functools.lru_cache(maxsize=256)
def _sequence_workspace_bytes(fp4, q_rows, requests, heads, kv_heads, head_dim, max_keys):
    lib = _lib.load()
    size = (lib.dsa_paged_attention_fp4_workspace_bytes if fp4
            else lib.dsa_seq_attention_workspace_bytes)
    return size(q_rows, requests, heads, kv_heads, head_dim, max_keys)


def _out_strides(q, out):
    """Strides of an attention's output, new (None) or given."""
    (rows, heads, head_dim), dtype = q[0], q[2]
    if out is None:
        return [heads * head_dim, head_dim]
    if out[0] != q[0] or out[2] != dtype:
        raise ValueError("out must have q's shape, type and device")
    _apart("out", out)
    strides = _row_strides(*out[:2], dtype.itemsize)
    if strides is None:
        if rows:
            raise ValueError("out must have a contiguous, 16-byte aligned head dimension")
        strides = [0, 0]
    return strides


@functools.lru_cache(maxsize=512)
def _attention_layout(paged, q, k, v, out):
    """(operands to copy first, strides, rows, heads, kv_heads, head_dim, dtype code) of a call."""
    code = dtype_code(q[2])
    dtype = q[2]
    if paged:
        keys = [_cache_strides("k_cache", k, dtype), _cache_strides("v_cache", v, dtype)]
        if k[0] != v[0] or len(q[0]) != 3 or k[0][3] != q[0][2]:
            raise ValueError("the caches must share their shape, and q [rows, heads, head_dim] "
                             "their head dimension")
        _page_size(k[0][1])
    else:
        keys = [_sequence_strides("k", k, dtype), _sequence_strides("v", v, dtype)]
        if k[0] != v[0] or len(q[0]) != 3 or k[0][2] != q[0][2]:
            raise ValueError("k and v must share their shape, and q [rows, heads, head_dim] their "
                             "head dimension")
    q_strides = _sequence_strides("q", q, dtype)
    rows, heads, head_dim = q[0]
    kv_heads = k[0][-2]
    if kv_heads == 0 or heads == 0 or heads % kv_heads:
        raise ValueError(f"{heads} query heads do not share {kv_heads} key/value heads")
    if head_dim % 8 or not 8 <= head_dim <= HEAD_DIM:
        raise ValueError(f"head_dim {head_dim} unsupported (a multiple of 8 up to {HEAD_DIM})")
    o_strides = _out_strides(q, out)
    every = [q_strides, *keys, o_strides]
    copies = tuple(i for i, x in enumerate(every) if x is None)
    strides = None if copies else (_I64x10 if paged else _I64x8)(*[x for t in every for x in t])
    return copies, strides, rows, heads, kv_heads, head_dim, code


def _sequence_buffers(q, layout, q_start, scale, out, return_lse, max_keys, fp4=False):
    """(scale, out, lse, workspace) of an attention call."""
    _, _, rows, heads, kv_heads, head_dim, _ = layout
    device = q.device
    scale = head_dim ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError(f"scale must be positive and finite, got {scale}")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        if out.device != device:
            raise ValueError("out must have q's shape, type and device")
        _aligned("out", out)
    lse = torch.empty((heads, rows), dtype=torch.float32, device=device) if return_lse else None
    workspace = torch.empty(
        _sequence_workspace_bytes(fp4, rows, q_start.shape[0] - 1, heads, kv_heads, head_dim,
                                  max_keys),
        dtype=torch.uint8, device=device)
    return scale, out, lse, workspace


def packed_attention(q, k, v, q_start, k_start=None, causal=True, scale=None, out=None,
                     return_lse=False):
    """Attention over sequences of different lengths packed side by side.

    q: [rows, heads, head_dim], k/v: [keys, kv_heads, head_dim], bf16 or fp16,
    head_dim a multiple of 8 up to 128, heads a multiple of kv_heads (query head
    h reads key/value head h // (heads / kv_heads)), any strides with a
    contiguous head dim.  Sequence r has the rows ``q_start[r]`` ..
    ``q_start[r + 1]`` of q and the same of k and v, or those of ``k_start``
    (int32 on the device, ascending).  ``causal``: of n rows and m keys row t
    attends to keys j <= t + m - n, so that the last row sees every key.  Lengths
    are read on the device only; a call of fewer sequences passes equal starts.

    Returns O [rows, heads, head_dim] (0 for rows that see no key) and, with
    ``return_lse``, the natural-log LSE [heads, rows] fp32 (-inf for those).  Rows
    outside every sequence are 0, or left as they were in a given ``out``, which
    may be q itself but overlaps no other operand and no other part of q.
    Forward only, as every attention here.
    """
    lib = _lib.load()
    _require_cuda("q", q)
    _require_cuda("k", k)
    _require_cuda("v", v)
    fill = out is None
    if not fill:
        _require_cuda("out", out)
    layout = _attention_layout(False, _layout(q), _layout(k), _layout(v),
                               None if fill else _layout(out))
    copies, strides, rows, heads, kv_heads, head_dim, code = layout
    device = q.device
    if not (k.device == v.device == device):
        raise ValueError("q, k and v must be on the same device")
    q_start = _index_vector("q_start", q_start, device)
    if q_start.shape[0] == 0:
        raise ValueError("q_start must hold one value more than there are sequences")
    requests = q_start.shape[0] - 1
    if k_start is not None:
        k_start = _index_vector("k_start", k_start, device, requests + 1)
    if copies or (q.data_ptr() | k.data_ptr() | v.data_ptr()) & 15:
        return packed_attention(*_in_place(copies, q, k, v), q_start, k_start, causal, scale, out,
                                return_lse)
    k_rows = k.shape[0]
    scale, out, lse, workspace = _sequence_buffers(q, layout, q_start, scale, out, return_lse,
                                                   k_rows)
    if rows:
        _call(lib.dsa_packed_attention, "dsa_packed_attention", device, q.data_ptr(),
              k.data_ptr(), v.data_ptr(), out.data_ptr(), code, strides, rows, k_rows, requests,
              heads, kv_heads, head_dim, q_start.data_ptr(),
              None if k_start is None else k_start.data_ptr(), scale, 1 if causal else 0,
              1 if fill else 0, None if lse is None else lse.data_ptr(), workspace.data_ptr(),
              workspace.shape[0])
    return (out, lse) if return_lse else out


def paged_attention(q, k_cache, v_cache, block_table, kv_lens, q_start, causal=True, scale=None,
                    out=None, return_lse=False):
    """Attention of new tokens over a paged key/value cache.

    q: [rows, heads, head_dim] as in ``packed_attention``; request r has the
    rows ``q_start[r]`` .. ``q_start[r + 1]`` and attends to the first
    ``kv_lens[r]`` tokens (its new ones, already written, included) of the pages
    in ``block_table[r]``.  One row per request is a decoding step, more are a
    chunk of a prompt or of a video's next frames; ``causal=False`` lets every
    row see every key.  k_cache, v_cache: [pages, page_size, kv_heads, head_dim],
    page_size a power of two from 16, read in place.  A table entry outside the
    cache takes no part: its keys are left out.  Returns as ``packed_attention``.
    """
    lib = _lib.load()
    _require_cuda("q", q)
    _require_cuda("k_cache", k_cache)
    _require_cuda("v_cache", v_cache)
    fill = out is None
    if not fill:
        _require_cuda("out", out)
    layout = _attention_layout(True, _layout(q), _layout(k_cache), _layout(v_cache),
                               None if fill else _layout(out))
    copies, strides, rows, heads, kv_heads, head_dim, code = layout
    device = q.device
    if not (k_cache.device == v_cache.device == device):
        raise ValueError("q and the caches must be on the same device")
    _aligned("k_cache", k_cache)
    _aligned("v_cache", v_cache)
    pages, page_size = k_cache.shape[:2]
    kv_lens = _index_vector("kv_lens", kv_lens, device)
    requests = kv_lens.shape[0]
    table, table_stride, width = _block_table(block_table, device, requests)
    q_start = _index_vector("q_start", q_start, device, requests + 1)
    if copies or q.data_ptr() & 15:
        return paged_attention(*_in_place(copies, q), k_cache, v_cache, block_table, kv_lens, q_start, causal,
                               scale, out, return_lse)
    scale, out, lse, workspace = _sequence_buffers(q, layout, q_start, scale, out, return_lse,
                                                   width * page_size)
    if rows:
        _call(lib.dsa_paged_attention, "dsa_paged_attention", device, q.data_ptr(),
              k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), code, strides, rows, requests,
              heads, kv_heads, head_dim, pages, page_size, table, table_stride, width,
              kv_lens.data_ptr(), q_start.data_ptr(), scale, 1 if causal else 0, 1 if fill else 0,
              None if lse is None else lse.data_ptr(), workspace.data_ptr(), workspace.shape[0])
    return (out, lse) if return_lse else out


# ---------------------------------------------------------------------------
# Writes that turn keys and queries with their positions; caches of 4-bit elements
# ---------------------------------------------------------------------------

def _fp4_row(head_dim):
    """Bytes of a token's keys and values in a 4-bit cache, for each key head."""
    if head_dim % 8 or not 8 <= head_dim <= HEAD_DIM:
        raise ValueError(f"head_dim {head_dim} unsupported (a multiple of 8 up to {HEAD_DIM})")
    return 32 * -(-head_dim // 32) + 8


def _fp4_page_size(value):
    _page_size(value)
    if value > 1 << 20:
        raise ValueError(f"page_size {value} unsupported for a 4-bit cache (up to 2^20)")


def paged_cache_fp4(pages, page_size, kv_heads, head_dim, device="cuda"):
    """An empty paged cache of 4-bit keys and values: uint8 [pages, kv_heads, page_size,
    32 * G + 8] with G = ceil(head_dim / 32): 4.25 bits an element at 128 dims, 4.5 at 64,
    and more where the last group is not full (5.2 at 80, 7.2 at 40, 20 at 8: more than 16
    bits).

    Groups of 32 neighbouring dims are E2M1 elements (0, 0.5, 1, 1.5, 2, 3, 4, 6 and
    their negatives) with a power of two between them.  The bytes of one page and head
    are, one after the other, the keys' codes [page_size, 16 * G], the values' codes,
    the keys' scale bytes [page_size, 4] and the values'; a scale byte b stands for
    2^(b - 127), 255 for a group that held an infinity or a NaN (and reads as NaN).
    Pages and heads may be any slices of a larger cache that are multiples of 16 bytes
    apart."""
    _fp4_page_size(page_size)
    if pages < 0 or kv_heads < 1:
        raise ValueError(f"a cache of {pages} pages of {kv_heads} key/value heads")
    return torch.zeros((pages, kv_heads, page_size, _fp4_row(head_dim)), dtype=torch.uint8,
                       device=device)


def _fp4_strides(layout, kv_heads, head_dim):
    """(page and head strides in bytes) of a 4-bit cache, used in place."""
    shape, strides, dtype = layout
    row = _fp4_row(head_dim)
    if dtype != torch.uint8 or len(shape) != 4 or shape[3] != row:
        raise ValueError(f"cache must be uint8 [pages, kv_heads, page_size, {row}] for "
                         f"{head_dim}-dim heads")
    if kv_heads is not None and shape[1] != kv_heads:
        raise ValueError(f"cache holds {shape[1]} key/value heads, not {kv_heads}")
    _fp4_page_size(shape[2])
    if strides[3] != 1 or strides[2] != row:
        raise ValueError("a page and head of the cache must be contiguous")
    lead = [0 if size == 1 else stride for size, stride in zip(shape[:2], strides[:2])]
    if any(stride % 16 for stride in lead):
        raise ValueError("pages and heads of the cache must be multiples of 16 bytes apart")
    return lead


def _fp4_aligned(cache):
    if cache.data_ptr() & 15 and cache.numel():
        raise ValueError("cache must be 16-byte aligned")


@functools.lru_cache(maxsize=512)
def _turn_layout(q, q_out, k, v, cache, v_cache, angles):
    """(operands to copy first, strides, tokens, heads, kv_heads, head_dim, rot_dim, dtype
    code, pages, page size) of a write that turns its rows; v_cache None: to 4 bits."""
    dtype = k[2]
    code = dtype_code(dtype)
    rows = [_sequence_strides("k", k, dtype), _sequence_strides("v", v, dtype)]
    tokens, kv_heads, head_dim = k[0]
    if v[0] != k[0]:
        raise ValueError("k and v must have the same shape")
    if kv_heads == 0:
        raise ValueError("k must hold at least one head")
    _fp4_row(head_dim)
    rot = 0
    if angles is not None:
        shape, own = angles
        if own != torch.float32 or len(shape) != 3 or shape[2] != 2:
            raise ValueError("cos_sin must be a float32 tensor [positions, rot_dim / 2, 2]")
        rot = 2 * shape[1]
        if rot % 16 or rot > head_dim:
            raise ValueError(f"{rot} turned dims unsupported (a multiple of 16 up to head_dim)")
        if shape[0] >= 1 << 31:
            raise ValueError("cos_sin must have fewer than 2^31 positions")
    heads, q_strides, out_strides = 0, [0, 0], [0, 0]
    if q is not None:
        q_strides = _sequence_strides("q", q, dtype)
        heads = q[0][1]
        if q[0] != (tokens, heads, head_dim):
            raise ValueError("q must have k's tokens and head dimension")
        out_strides = [heads * head_dim, head_dim]
        if q_out is not None:
            if q_out[0] != q[0] or q_out[2] != dtype:
                raise ValueError("q_out must have q's shape, type and device")
            _apart("q_out", q_out)
            out_strides = _row_strides(*q_out[:2], dtype.itemsize)
            if out_strides is None:
                if tokens and heads:
                    raise ValueError("q_out must have a contiguous, 16-byte aligned head dimension")
                out_strides = [0, 0]
    if v_cache is None:
        held = [_fp4_strides(cache, kv_heads, head_dim)]
        pages, _, page_size, _ = cache[0]
        _apart("cache", cache)
    else:
        held = [_cache_strides("k_cache", cache, dtype), _cache_strides("v_cache", v_cache, dtype)]
        pages, page_size = cache[0][:2]
        if cache[0] != v_cache[0] or cache[0][2:] != (kv_heads, head_dim):
            raise ValueError("the caches must share their shape, and k its heads and head "
                             "dimension")
        _page_size(page_size)
        _apart("k_cache", cache)
        _apart("v_cache", v_cache)
    operands = [q_strides, out_strides, *rows, *held]
    copies = tuple(i for i, x in enumerate((q_strides, *rows)) if x is None)
    strides = None
    if not copies:
        strides = (_I64x10 if v_cache is None else _I64x14)(*[x for t in operands for x in t])
    return copies, strides, tokens, heads, kv_heads, head_dim, rot, code, pages, page_size


def _on_device(name, t, device):
    """Refuses what is not a tensor on the call's (HIP) device."""
    if not isinstance(t, torch.Tensor) or t.device != device:
        _require_cuda(name, t)
        raise ValueError(f"{name} must live on {device}")


def _write_turned(function, what, k, v, caches, slots, positions, cos_sin, q, q_out, halves):
    """A write of both kinds; returns the turned queries, or None."""
    device = caches[0].device
    try:
        here = (k.device == device and v.device == device and slots.device == device
                and (q is None or q.device == device))
    except AttributeError:
        here = False
    if not here:
        for name, t in (("k", k), ("v", v), ("slots", slots), ("q", q)):
            if t is not None or name != "q":
                _on_device(name, t, device)
    if q_out is not None:
        _on_device("q_out", q_out, device)
        if q is None:
            raise ValueError("q_out needs q")
    copies, strides, tokens, heads, kv_heads, head_dim, rot, code, pages, page_size = _turn_layout(
        None if q is None else _layout(q), None if q_out is None else _layout(q_out), _layout(k),
        _layout(v), _layout(caches[0]), _layout(caches[1]) if len(caches) > 1 else None,
        None if cos_sin is None else (cos_sin.shape, cos_sin.dtype))
    if slots.dtype != torch.int64 or slots.shape != (tokens,):
        raise ValueError(f"slots must be an int64 tensor of {tokens} values")
    if not slots.is_contiguous():
        slots = slots.contiguous()
    angles = turns = None
    if cos_sin is not None:
        _on_device("cos_sin", cos_sin, device)
        positions = _index_vector("positions", positions, device, tokens)
        if not cos_sin.is_contiguous() or cos_sin.data_ptr() & 15:
            cos_sin = cos_sin.clone(memory_format=torch.contiguous_format)
        if rot:
            turns, angles = positions.data_ptr(), cos_sin.data_ptr()
    elif positions is not None:
        raise ValueError("positions need cos_sin")
    at_q, at_k, at_v = 0 if q is None else q.data_ptr(), k.data_ptr(), v.data_ptr()
    if copies or (at_q | at_k | at_v) & 15:
        # (a copied q still goes to its own place where q_out is q)
        new_q, k, v = _in_place(copies, k if q is None else q, k, v)
        return _write_turned(function, what, k, v, caches, slots, positions, cos_sin,
                             None if q is None else new_q, q_out, halves)
    out, at_out = q_out, 0
    if q is not None:
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        else:
            _aligned("q_out", out)
        at_out = out.data_ptr()
    if tokens:
        first = caches[0].data_ptr()
        held = (first,) if len(caches) == 1 else (first, caches[1].data_ptr())
        _call(function, what, device, at_q, at_out, at_k, at_v, *held, code, strides, tokens, heads,
              kv_heads, head_dim, rot, 1 if halves else 0, pages, page_size, slots.data_ptr(), turns,
              angles, cos_sin.shape[0] if rot else 0)
    return out


def paged_write_rotary(k, v, k_cache, v_cache, slots, positions, cos_sin, q=None, q_out=None,
                       halves=False):
    """``paged_write`` that turns the keys with their positions on the way, and the
    queries beside them.

    cos_sin: float32 [positions, rot_dim / 2, 2] on the device, (cos, sin) of every
    position's angles (as ``rmsnorm_rope`` takes them); the first rot_dim dims of a
    head, a multiple of 16, turn in neighbouring pairs (2 i, 2 i + 1) or, with
    ``halves``, in pairs (i, i + rot_dim / 2).  positions: int32 [tokens] on the device,
    the rows of cos_sin.  A step's, behind its plan and with nothing read back::

        token = torch.arange(tokens, device=device)
        r = torch.searchsorted(plan.q_start[1:], token, right=True).clamp_max(requests - 1)
        positions = (cached[r] + token - plan.q_start[r]).int()

    k, v, the caches and slots as in ``paged_write``, bf16 or fp16, head_dim a multiple
    of 8 up to 128; a token whose position is outside cos_sin is skipped as one without
    a slot.  q [tokens, heads, head_dim] (optional): returned turned, in a new tensor or
    in ``q_out``, which may be q itself; a row whose position is outside cos_sin is
    passed on as it is.  Elements are turned in float32 and rounded once.
    """
    lib = _lib.load()
    _require_cuda("k_cache", k_cache)
    _on_device("v_cache", v_cache, k_cache.device)
    _aligned("k_cache", k_cache)
    _aligned("v_cache", v_cache)
    if cos_sin is None:
        raise ValueError("cos_sin and positions are needed (paged_write turns nothing)")
    return _write_turned(lib.dsa_paged_write_rotary, "dsa_paged_write_rotary", k, v,
                         (k_cache, v_cache), slots, positions, cos_sin, q, q_out, halves)


def paged_write_fp4(k, v, cache, slots, positions=None, cos_sin=None, q=None, q_out=None,
                    halves=False):
    """Writes keys and values [tokens, kv_heads, head_dim] (bf16 or fp16) into a cache of
    4-bit elements (``paged_cache_fp4``), row t at slot ``slots[t]``.

    With ``cos_sin`` and ``positions`` the keys (and q) turn first, as in
    ``paged_write_rotary``; the rest of its conditions hold here too.  Each group of 32
    neighbouring dims gets the smallest exponent e with max|x| <= 7 * 2^e, between -125
    and 125 (fp16: -23 and 13, so that every element is a number of that type; larger
    elements become the largest), and its elements the nearest codes, ties the even
    ones, from the turned value in float32.  Normal values are off by 11% of their norm.
    A group with an infinity or a NaN is kept as NaN.  Returns q turned (without
    cos_sin: as it is), or None.
    """
    lib = _lib.load()
    _require_cuda("cache", cache)
    _fp4_aligned(cache)
    return _write_turned(lib.dsa_paged_write_fp4, "dsa_paged_write_fp4", k, v, (cache,), slots,
                         positions, cos_sin, q, q_out, halves)


@functools.lru_cache(maxsize=512)
def _read_layout(cache, head_dim, dtype):
    """(dtype code, strides, pages, key heads, page size) of a read."""
    code = dtype_code(dtype)
    strides = _I64x2(*_fp4_strides(cache, None, head_dim))
    pages, kv_heads, page_size, _ = cache[0]
    return code, strides, pages, kv_heads, page_size


def paged_read_fp4(cache, head_dim, pages=None, dtype=torch.bfloat16):
    """Keys and values that a 4-bit cache stands for, (k, v) [pages, page_size, kv_heads,
    head_dim] in bf16 or fp16: of the listed ``pages`` (int32 on the device, zeros for
    one outside the cache) or of all.  Exact, but for elements that fp16 cannot hold of a
    cache written from bf16."""
    lib = _lib.load()
    _require_cuda("cache", cache)
    code, strides, total, kv_heads, page_size = _read_layout(_layout(cache), head_dim, dtype)
    _fp4_aligned(cache)
    device = cache.device
    if pages is not None:
        pages = _index_vector("pages", pages, device)
    count = total if pages is None else pages.shape[0]
    shape = (count, page_size, kv_heads, head_dim)
    k = torch.empty(shape, dtype=dtype, device=device)
    v = torch.empty_like(k)
    if count and kv_heads:
        _call(lib.dsa_paged_read_fp4, "dsa_paged_read_fp4", device, cache.data_ptr(), strides,
              k.data_ptr(), v.data_ptr(), code, total, page_size, kv_heads, head_dim,
              None if pages is None else pages.data_ptr(), count)
    return k, v


@functools.lru_cache(maxsize=512)
def _fp4_attention_layout(q, cache, out):
    """As ``_attention_layout`` over a 4-bit cache."""
    dtype = q[2]
    code = dtype_code(dtype)
    q_strides = _sequence_strides("q", q, dtype)
    rows, heads, head_dim = q[0]
    held = _fp4_strides(cache, None, head_dim)
    kv_heads = cache[0][1]
    if kv_heads == 0 or heads == 0 or heads % kv_heads:
        raise ValueError(f"{heads} query heads do not share {kv_heads} key/value heads")
    o_strides = _out_strides(q, out)
    copies = () if q_strides is not None else (0,)
    strides = None if copies else _I64x6(*q_strides, *held, *o_strides)
    return copies, strides, rows, heads, kv_heads, head_dim, code


def paged_attention_fp4(q, cache, block_table, kv_lens, q_start, causal=True, scale=None, out=None,
                        return_lse=False):
    """``paged_attention`` over a cache of 4-bit elements (``paged_cache_fp4``).

    The keys and values are those that ``paged_read_fp4`` gives in q's type, read in
    place: a decoding step reads 27% of a 16-bit cache's bytes.  q's type is the one
    that the cache was written from.  Everything else, and what is returned, as in
    ``paged_attention``, its precision too: scores and sums in float32, the probabilities
    rounded to q's type before they meet V.  A group of 32 dims that is not a number (``paged_write_fp4``)
    makes the rows that see its key NaN, one of values those dims of them; so does, with
    fp16 queries over a cache written from bf16, a group of values past 57,344, which has
    elements that fp16 cannot hold.
    """
    lib = _lib.load()
    _require_cuda("q", q)
    _require_cuda("cache", cache)
    fill = out is None
    if not fill:
        _require_cuda("out", out)
    layout = _fp4_attention_layout(_layout(q), _layout(cache), None if fill else _layout(out))
    copies, strides, rows, heads, kv_heads, head_dim, code = layout
    device = q.device
    if cache.device != device:
        raise ValueError("q and the cache must be on the same device")
    _fp4_aligned(cache)
    pages, _, page_size, _ = cache.shape
    kv_lens = _index_vector("kv_lens", kv_lens, device)
    requests = kv_lens.shape[0]
    table, table_stride, width = _block_table(block_table, device, requests)
    q_start = _index_vector("q_start", q_start, device, requests + 1)
    if copies or q.data_ptr() & 15:
        return paged_attention_fp4(*_in_place(copies, q), cache, block_table, kv_lens, q_start,
                                   causal, scale, out, return_lse)
    scale, out, lse, workspace = _sequence_buffers(q, layout, q_start, scale, out, return_lse,
                                                   width * page_size, fp4=True)
    if rows:
        _call(lib.dsa_paged_attention_fp4, "dsa_paged_attention_fp4", device, q.data_ptr(),
              cache.data_ptr(), out.data_ptr(), code, strides, rows, requests, heads, kv_heads,
              head_dim, pages, page_size, table, table_stride, width, kv_lens.data_ptr(),
              q_start.data_ptr(), scale, 1 if causal else 0, 1 if fill else 0,
              None if lse is None else lse.data_ptr(), workspace.data_ptr(), workspace.shape[0])
    return (out, lse) if return_lse else out
