"""Low-rank adapters of several requests beside one shared projection.

``low_rank`` adds scale[a] * up[a] (down[a] x) to a projection's output, with
the adapter a chosen per sequence or per row, so that one batch serves
requests with different adapters over one (bf16 or MXFP8) weight.  The
reference has no adapters; there is no reference counterpart.  Kernels:
libqim's ``qim_low_rank``.
"""
import torch

from qwen_image_accel import _native

MAX_RANK = 128


def _rows(t):
    """(rows, width, row stride) of a (M, W) or (B, S, W) tensor whose rows lie
    one stride apart, else None.  An axis of one element may have any stride."""
    shape = t.shape
    if len(shape) not in (2, 3):
        return None
    w = shape[-1]
    rows = shape[0] if len(shape) == 2 else shape[0] * shape[1]
    if t.is_contiguous():
        return rows, w, w
    if w > 1 and t.stride(-1) != 1:
        return None
    if len(shape) == 2:
        return rows, w, t.stride(0) if rows > 1 else w
    b, s = shape[:2]
    row = t.stride(1) if s > 1 else t.stride(0) if b > 1 else w
    if b > 1 and s > 1 and t.stride(0) != s * row:
        return None
    return rows, w, row


def takes_rows(t):
    """Whether ``low_rank`` takes the rows of t as they lie: one multiple of 8
    elements apart, 16-byte aligned."""
    rows = _rows(t)
    return rows is not None and rows[2] >= rows[1] and rows[2] % 8 == 0 and t.data_ptr() % 16 == 0


def low_rank(x, down, up, index, *, scale=None, base=None, out=None, parts=1):
    """``base + scale[a] * (x @ down[a].T) @ up[a].T`` per row, a = ``index``.

    x: (M, K) or (B, S, K) bf16.  down: (A, parts * R, K) and up: (A, N, R)
    bf16, R <= 128.  ``index``: int32 on the GPU, (M,) for (M, K), one per row,
    or (B,) for (B, S, K), one per sequence; a row whose entry is outside
    [0, A) (-1 by convention) has no adapter.  ``scale``: None or fp32 (A,).
    ``base``: the projection's output, (M, N) or (B, S, N) bf16, or None
    (zeros); ``out``: where the result goes, by default a new tensor; ``base`` itself is fine, else it
    shares no rows with ``base`` or ``x``.
    ``parts``: N is that many equal column blocks, and block j uses rows
    [j * R, (j + 1) * R) of down: the adapters of a stacked projection (Q/K/V)
    in one call.  The sum is taken in fp32 and rounded once.  K, R and
    N / parts are multiples of 8; rows may lie any multiple of 8 elements apart.
    No value of another row enters a row.  Its bits are the same for the same number
    of rows and sequence length; another of these may order the fp32 sums differently.
    No gradient is recorded."""
    def refuse(why):
        raise _native.Unsupported("low_rank", _native.QIM_ERR_LAYOUT, why)
    device = x.device
    if not x.is_cuda:
        refuse("expects tensors on the GPU")
    xr = _rows(x)
    bf16, lead = torch.bfloat16, x.shape[:-1]
    if x.dtype != bf16 or xr is None or xr[1] == 0:
        refuse("x is a bf16 (M, K) or (B, S, K) tensor, K > 0, with rows one stride apart")
    m, k, ldx = xr
    if (up.dim() != 3 or down.dtype != bf16 or up.dtype != bf16 or parts < 1
            or down.shape != (up.shape[0], parts * up.shape[2], k) or not down.is_contiguous() or not up.is_contiguous()
            or down.device != device or up.device != device):
        refuse(f"down (A, {parts} * R, {k}) and up (A, N, R) are contiguous bf16 tensors on {device}")
    a, n, r = up.shape
    if index.dtype != torch.int32 or index.device != device or index.shape != lead[:1] or not index.is_contiguous():
        refuse(f"index is a contiguous int32 ({x.shape[0]},) tensor on {device}")
    if scale is not None and (scale.dtype != torch.float32 or scale.shape != (a,) or scale.device != device
                              or not scale.is_contiguous()):
        refuse(f"scale is a contiguous fp32 ({a},) tensor on {device}")
    shape = lead + (n,)

    def stride(t):
        rows = _rows(t)
        if rows is None or t.dtype != bf16 or t.shape != shape or t.device != device:
            refuse(f"base and out are bf16 {tuple(shape)} tensors on {device} with rows one stride apart")
        return rows[2]
    ldb = 0 if base is None else stride(base)
    if out is None:
        out, ldo = torch.empty(shape, dtype=bf16, device=device), n
    else:
        ldo = ldb if out is base else stride(out)
    if m == 0 or n == 0:
        return out
    seq = lead[1] if len(lead) == 2 else 1
    nbytes = _native.bytes_on(device, "qim_low_rank_workspace_bytes", m, seq, k, r, parts)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    _native.call_on(device, "qim_low_rank", x.data_ptr(), ldx, down.data_ptr(), up.data_ptr(), index.data_ptr(),
                    _native.ptr(scale), _native.ptr(base), ldb, out.data_ptr(), ldo, _native.ptr(ws), nbytes,
                    m, seq, k, n, r, parts, a)
    return out
