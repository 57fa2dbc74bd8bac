"""Thin torch-facing wrappers: pass data_ptr()s and the current stream to the C ABI.

Host-side mirror of the reference's packers and launch wrappers:
  _pack                 thunderworld_fp4/linear.py:13-25
  pack (calibrated)     thunderworld_fp4/_calibrated.py:60-71
  pack_sparse           thunderworld_fp4/_sparse_pack.py:77-93
  pack_with_factor      thunderworld_fp4/_fusion.py:37-42
  pack_input / swizzle  thunderworld_fp4/cutlass/packing.py:85-109, cutlass/layout.py:16-25
  CutlassFused.run_packed  thunderworld_fp4/cutlass/backend.py:48-71
torch is used for device memory and streams only.
"""
import ctypes
import threading
from contextlib import nullcontext
from dataclasses import dataclass
from functools import lru_cache
import torch
from . import _lib


def cdiv(a, b):
    return (a + b - 1) // b


_checked_devices = set()          # a device's capability does not change: asked once


def require_sm100(device):
    if device in _checked_devices:
        return
    if device.type != 'cuda':
        raise ValueError('a CUDA device is required')
    if torch.cuda.get_device_capability(device)[0] != 10:
        raise RuntimeError('thunderworld_b200 kernels are built for sm_100a (B200) only; no fallback exists')
    if device.index is not None:
        _checked_devices.add(device)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream(device):
    # the raw handle, without the Stream object that torch.cuda.current_stream makes (2.2 us of a small call's 25)
    if device.index is None:
        return torch.cuda.current_stream(device).cuda_stream
    return torch._C._cuda_getCurrentRawStream(device.index)


_same_device = nullcontext()


def _device(device):
    """Context that makes `device` current; nothing to do, and nothing done, when it is."""
    return _same_device if torch.cuda.current_device() == device.index else torch.cuda.device(device)


# Scratch per stream: calls on one stream run one after the other. A call that is being captured gets scratch of its own graph's, so
# that two graphs captured on one stream may be replayed side by side; only the newest capture's is held here, older ones live as
# long as their graph's pool. 'zeroed' is 8 bytes that kernels leave zeroed (the graph zeroes its own on every replay), 'paged'
# needs no initialisation and grows as wanted. A call of two launches has its plan in the scratch between them, so threads take turns
# from the lookup to the last launch (`_launching`; ctypes lets other threads run meanwhile).
_stream_scratch = {}
_launching, _making = threading.Lock(), threading.Lock()


def _scratch(device, stream, kind='zeroed', nbytes=8):
    capture = _lib.load().tw_capture_id(stream)
    key = (device, stream, kind, capture != 0)
    held = _stream_scratch.get(key)
    if held is None or held[0] != capture or held[1].numel() < nbytes:
        with _making:                                             # two threads that both find none share one
            held = _stream_scratch.get(key)
            if held is None or held[0] != capture or held[1].numel() < nbytes:
                make = torch.zeros if kind == 'zeroed' else torch.empty
                held = _stream_scratch[key] = (capture, make(nbytes, device=device, dtype=torch.uint8))
    return held[1]


@dataclass
class Packed:
    """Quantized activation: the reference's (codes, scales, factor, mp) tuple plus the atom-layout
    scales and alpha that the fused GEMM reads (reference: cutlass/packing.py CutlassPacked)."""
    codes: torch.Tensor          # uint8 [planes, mp, k/2]
    scales: torch.Tensor         # float8_e4m3fn [planes, mp, k/16]
    factor: torch.Tensor         # float32 scalar
    mp: int
    scales_swz: torch.Tensor     # uint8 [planes, ceil(m/128)*128, k/16] atom layout
    alpha: torch.Tensor          # float32 scalar = factor * wg (when wg was given)
    mask: torch.Tensor           # bool [ceil(m/128), k/128] or None

    @property
    def native(self):
        return self.codes, self.scales, self.factor, self.mp

    def __iter__(self):          # unpack like the reference tuple
        return iter(self.native)


# One scratch buffer per device and kernel family, shared by every call: like the reference engine,
# callers issue one request at a time on one stream (docs/INFERENCE.md:51 of the reference).
_workspaces = {}


def _workspace(device, nbytes, key):
    ws = _workspaces.get((device, key))
    if ws is None or ws.numel() < nbytes:
        with torch.inference_mode(False):                 # reset_device_status writes to it outside of that mode as well
            ws = torch.zeros(max(nbytes, 256), device=device, dtype=torch.uint8)
        _workspaces[(device, key)] = ws
    return ws


def quantize(x, prescale=None, *, repair=1, mask=None, na=0, sensitivity=None, factor=None, wg=None,
             base=1., res=1., gain=1., energy=1., workspace=None, out=None):
    """bf16 [m,k] -> Packed. repair: 0 base only, 1 full residual, 2 residual under `mask`,
    3 online selection of `na` K128 blocks per M128 row block (mask is written)."""
    if x.ndim != 2 or x.dtype != torch.bfloat16 or not x.is_contiguous():
        raise ValueError('expected contiguous BF16 [M,K]')
    require_sm100(x.device)
    m, k = x.shape
    if m == 0:
        raise ValueError('empty activation rows are unsupported')
    if k % 128:
        raise ValueError('K must be a multiple of 128')
    lib = _lib.load()
    # with preallocated outputs the planes may hold more rows than m (a shard of a larger gathered tensor)
    mp = cdiv(m, 16) * 16 if out is None else int(out.codes.shape[1])
    mb = cdiv(m, 128)
    if mp < cdiv(m, 16) * 16:
        raise ValueError('preallocated planes are too small')
    planes = 2 if repair else 1
    dev = x.device
    if out is None:
        codes = torch.empty((planes, mp, k // 2), device=dev, dtype=torch.uint8)
        scales = torch.empty((planes, mp, k // 16), device=dev, dtype=torch.float8_e4m3fn)
        swz = torch.empty((planes, mb * 128, k // 16), device=dev, dtype=torch.uint8)
        fac = torch.empty((), device=dev, dtype=torch.float32) if factor is None else factor
        alpha = torch.empty((), device=dev, dtype=torch.float32)
        if repair == 3 and mask is None:
            mask = torch.empty((mb, k // 128), device=dev, dtype=torch.bool)
    else:
        codes, scales, swz, fac, alpha = out.codes, out.scales, out.scales_swz, out.factor, out.alpha
        mask = out.mask if mask is None else mask
    if repair in (2, 3) and (mask is None or mask.dtype != torch.bool or tuple(mask.shape) != (mb, k // 128)
                             or not mask.is_contiguous()):
        raise ValueError(f'mask must be contiguous bool {(mb, k // 128)}')
    if workspace is None:
        workspace = _workspace(dev, lib.tw_quantize_workspace(m, k), 'q')
    args = _lib.QuantizeArgs(_ptr(x), _ptr(prescale), _ptr(sensitivity), _ptr(fac), _ptr(wg), _ptr(alpha),
                             _ptr(codes), _ptr(scales), _ptr(swz), _ptr(mask), _ptr(workspace),
                             m, k, mp, int(repair), int(na), int(factor is not None),
                             float(base), float(res), float(gain), float(energy), int(swz.shape[1]))
    with torch.cuda.device(dev):
        _lib.check(lib.tw_quantize(ctypes.byref(args), _stream(dev)))
    return Packed(codes, scales, fac, mp, swz, alpha, mask)


def swizzle(scales):
    """Row-major E4M3 [rows, cols] -> atom layout uint8 [ceil(rows/128)*128, cols]."""
    if scales.dtype not in (torch.float8_e4m3fn, torch.uint8) or not scales.is_contiguous() or scales.ndim != 2:
        raise ValueError('Contiguous E4M3 scales required')
    rows, cols = scales.shape
    if cols % 4:
        raise ValueError('Scale columns must be divisible by four')
    require_sm100(scales.device)
    out = torch.empty((cdiv(rows, 128) * 128, cols), device=scales.device, dtype=torch.uint8)
    with torch.cuda.device(scales.device):
        _lib.check(_lib.load().tw_swizzle_scales(scales.data_ptr(), rows, cols, out.data_ptr(), _stream(scales.device)))
    return out


def activation_rank(x, prescale=None):
    """int32 [ceil(m/128), k/128]: rank of every K128 block within its M128 row block by sampled energy
    (reference: activation_rank, thunderworld_fp4/_linear_kernels.py:23-34). One launch, no host sync."""
    if x.ndim != 2 or x.dtype != torch.bfloat16 or not x.is_contiguous() or x.shape[1] % 128 or x.shape[0] == 0:
        raise ValueError('expected contiguous BF16 [M,K] with K a multiple of 128')
    require_sm100(x.device)
    m, k = x.shape
    rank = torch.empty((cdiv(m, 128), k // 128), device=x.device, dtype=torch.int32)
    with torch.cuda.device(x.device):
        _lib.check(_lib.load().tw_activation_rank(_ptr(x), _ptr(prescale), m, k, _ptr(rank), _stream(x.device)))
    return rank


def selftest_bounded_wait(device=None, limit_cycles=2_000_000):
    """Make a bounded device-side wait run out on purpose (a barrier nothing signals) and return the status word
    that `device_status` then reports; the word is left set so that the caller can see and reset it."""
    dev = torch.device('cuda', torch.cuda.current_device()) if device is None else torch.device(device)
    ws = _workspace(dev, 256, 'g')
    with torch.cuda.device(dev):
        _lib.check(_lib.load().tw_selftest_bounded_wait(_ptr(ws), int(limit_cycles), _stream(dev)))
    return device_status(dev)


def fused_gemm(m, n, k, packed, wc, ws_swz, alpha, *, na=0, mask=None, wr=None, wrs_swz=None, wi=None, off=None,
               wloc=None, cross=False, shared=False, dense=False, ws=None, wrs=None, out=None, workspace=None,
               mask_per_n=False, bias=None, kernel=0, activation=None, want_stats=False):
    """One launch of the repaired GEMM; returns bf16 [m,n]. activation='gelu_tanh' applies the activation to the
    bf16-rounded result in the epilogue (the bits activate_with_factor would give); with want_stats the call returns
    (out, stats) with stats = float32 [2] = (max|out| / 2688, max|out|)."""
    lib = _lib.load()
    dev = wc.device
    require_sm100(dev)
    if out is None:
        out = torch.empty((m, n), device=dev, dtype=torch.bfloat16)
    if workspace is None:
        workspace = _workspace(dev, lib.tw_workspace(m, n, k), 'g')
    hasw = wr is not None and wr.numel() > 0
    a0s = packed.scales_swz[0]
    a1s = packed.scales_swz[1] if packed.scales_swz.shape[0] > 1 else None
    io = _lib.RepairIO(_ptr(packed.codes), _ptr(packed.scales), _ptr(wc), _ptr(ws), _ptr(wr) if hasw else None,
                       _ptr(wrs) if hasw else None, _ptr(wi), _ptr(off), _ptr(wloc), _ptr(mask),
                       m, packed.mp, n, k, int(na), int(hasw), int(cross), int(shared), int(dense),
                       int(wr.shape[0]) if hasw else 0, _ptr(a1s) if na else None, _ptr(wrs_swz) if hasw else None,
                       _ptr(bias), int(mask_per_n), int(kernel), 0, None, None)
    stats = None
    if activation is not None:
        if activation != 'gelu_tanh':
            raise ValueError('the GEMM epilogue fuses gelu_tanh only')
        io.activation = ACT_MODES[activation]
        if want_stats:
            stats, scratch = _stats(dev, True)
            io.stats, io.stats_scratch = _ptr(stats), _ptr(scratch)
    elif want_stats:
        raise ValueError('stats come with a fused activation')
    with torch.cuda.device(dev):
        _lib.check(lib.tw_fused(m, n, k, packed.codes.data_ptr(), wc.data_ptr(), a0s.data_ptr(), ws_swz.data_ptr(),
                                out.data_ptr(), alpha.data_ptr(), workspace.data_ptr(), _stream(dev), ctypes.byref(io)))
    return (out, stats) if want_stats else out


MATVEC_ROWS = 32


def fp4_matvec(x, codes, scales, factor, *, prescale=None, bias=None, wr=None, wrs=None, wi=None, off=None, wloc=None,
               shared=False, dense=False, out_dtype=torch.bfloat16, out=None):
    """Product of a few rows (at most 32) with packed NVFP4 weights, for a token at a time: x bf16 [..., K] stays bf16.

    y = factor * (bf16(x * prescale) @ W.T) + bias, W = codes [N, K/2] x E4M3 scales [N, K/16] plus the W1 tiles of a bank
    (wr [slots, 128, 64], wrs [slots, 128, 8]; wi, off, wloc, shared, dense as in fused_gemm), sums of 32 bits, one rounding. Of a row,
    values below 2^-29 of the largest are held to within 2^-39 of the largest, all others exactly.
    factor: float32 scalar tensor; prescale float32 [K]; bias bf16 [N]; out_dtype bfloat16 or float32; out shares no memory with x. Any
    N, K a multiple of 32 up to 32768; with a bank both multiples of 128. One launch; where the rows' part of K does not fit an SM's
    shared memory (more than 29 rows of a K of 16384, 21 of 24576, 16 of 32768, with a bank 28, 20, 15) two or three, a share of the rows each."""
    if x.ndim < 1 or x.dtype is not torch.bfloat16 or not x.is_cuda:
        raise ValueError('expected CUDA BF16 rows [..., K]')
    if codes.ndim != 2 or codes.dtype is not torch.uint8 or not codes.is_contiguous():
        raise ValueError('codes must be contiguous uint8 [N,K/2]')
    n, k = codes.shape[0], codes.shape[1] * 2
    dev = x.device
    if x.shape[-1] != k:
        raise ValueError(f'expected {k} values per row')
    if tuple(scales.shape) != (n, k // 16) or scales.dtype is not torch.float8_e4m3fn or not scales.is_contiguous():
        raise ValueError('scales must be contiguous E4M3 [N,K/16]')
    if factor.dtype is not torch.float32 or factor.numel() != 1:
        raise ValueError('factor must be one float32 value')
    if prescale is not None and (tuple(prescale.shape) != (k,) or prescale.dtype is not torch.float32 or not prescale.is_contiguous()):
        raise ValueError('prescale must be contiguous float32 [K]')
    if bias is not None and (tuple(bias.shape) != (n,) or bias.dtype is not torch.bfloat16 or not bias.is_contiguous()):
        raise ValueError('bias must be contiguous BF16 [N]')
    if out_dtype is not torch.bfloat16 and out_dtype is not torch.float32:
        raise ValueError('out_dtype must be bfloat16 or float32')
    rows = x.numel() // k if k else 0
    if not rows or not n:
        raise ValueError('empty activation rows or weights are unsupported')
    if rows > MATVEC_ROWS:
        raise ValueError(f'at most {MATVEC_ROWS} rows; more go through the quantizer and fused_gemm')
    if torch.is_grad_enabled() and x.requires_grad:
        raise RuntimeError('fp4_matvec is inference-only; use torch.inference_mode()')
    slots = 0 if wr is None or (wi is not None and not dense and not wi.numel()) else wr.shape[0]     # a bank without an entry adds nothing
    if slots:
        if n % 128 or k % 128:
            raise ValueError('a W1 bank needs N and K to be multiples of 128')
        if tuple(wr.shape) != (slots, 128, 64) or wr.dtype is not torch.uint8 or not wr.is_contiguous():
            raise ValueError('wr must be contiguous uint8 [slots,128,64]')
        if wrs is None or wrs.numel() != slots * 1024 or wrs.element_size() != 1 or not wrs.is_contiguous():
            raise ValueError('wrs must be contiguous E4M3 [slots,128,8]')
        if not dense:
            for t, name in ((wi, 'wi'), (off, 'off')) + (((wloc, 'wloc'),) if shared else ()):
                if t is None or t.dtype is not torch.int32 or not t.is_contiguous():
                    raise ValueError(f'{name} must be contiguous int32')
            if off.numel() != n // 128 + 1 or (shared and wloc.numel() != wi.numel()):
                raise ValueError('off must hold N/128 + 1 offsets and wloc one position per entry of wi')
    for t in (codes, scales, factor, prescale, bias, wr, wrs, wi, off, wloc):
        if t is not None and t.device != dev:
            raise ValueError('activation and packed weights must share a CUDA device')
    require_sm100(dev)
    flat = x if x.ndim == 2 else x.reshape(-1, k)
    if flat.stride(1) != 1 or (rows > 1 and flat.stride(0) % 8) or flat.data_ptr() % 16:
        flat = flat.clone(memory_format=torch.contiguous_format)
    if prescale is not None and prescale.data_ptr() % 16:
        prescale = prescale.clone()
    shape = (*x.shape[:-1], n)
    if out is None:
        out = x.new_empty(shape, dtype=out_dtype)
    elif tuple(out.shape) != shape or out.dtype is not out_dtype or not out.is_contiguous() or out.device != dev:
        raise ValueError(f'out must be contiguous {out_dtype} {shape} on the device of x')
    elif _meet(_span(out), _span(flat)):
        raise ValueError('out must not share memory with x')
    args = _lib.MatvecArgs(flat.data_ptr(), flat.stride(0) if rows > 1 else k, _ptr(prescale), codes.data_ptr(), scales.data_ptr(),
                           factor.data_ptr(), _ptr(bias), _ptr(wr) if slots else None, _ptr(wrs) if slots else None, _ptr(wi),
                           _ptr(off), _ptr(wloc), out.data_ptr(), rows, n, k, slots, 0 if wi is None else wi.numel(),
                           int(shared), int(dense), int(out_dtype is torch.float32))
    with _device(dev):
        _lib.check(_lib.load().tw_matvec(ctypes.byref(args), _stream(dev)))
    return out


# ---- paged key-value cache --------------------------------------------------------------------------
_status_words = {}


def _cache_status(device):
    """Address of the device word that the paged operators report in (device_status reads it; it lives as long as the process)."""
    word = _status_words.get(device)
    if word is None:
        with _making:
            word = _status_words.get(device)
            if word is None:
                with _device(device):
                    if torch.cuda.is_current_stream_capturing():          # the word would be the graph's, and zero at every replay
                        raise RuntimeError('the first call of a paged operator on a device cannot be captured: make a PagedCache or call one before')
                    word = _workspace(device, 256, 'c').data_ptr()
                    torch.cuda.current_stream(device).synchronize()       # zeroed before another stream's call may write it
                _status_words[device] = word
    return word


def _check_pages(k_pages, v_pages):
    """(pages, kv heads, page, dim, fp8, strides of k, of v) of the two halves of a pool; raises where they are not pages."""
    shape, dtype = k_pages.shape, k_pages.dtype
    if len(shape) != 4 or shape != v_pages.shape or not k_pages.numel():
        raise ValueError('k_pages and v_pages must be [pages, kv_heads, page, dim] alike')
    if dtype is not v_pages.dtype or (dtype is not torch.bfloat16 and dtype is not torch.float8_e4m3fn):
        raise ValueError('pages must be bfloat16 or float8_e4m3fn')
    pages, hk, page, dim = shape
    if dim != 64 and dim != 128:
        raise ValueError('head dimension must be 64 or 128')
    if page & (page - 1):
        raise ValueError('tokens per page must be a power of two')
    ks, vs = k_pages.stride(), v_pages.stride()
    if ks[3] != 1 or vs[3] != 1 or (page > 1 and (ks[2] != dim or vs[2] != dim)):
        raise ValueError('the rows of a page must lie one behind the other')
    if not k_pages.is_cuda or v_pages.device != k_pages.device:
        raise ValueError('pages must be on one CUDA device')
    return pages, hk, page, dim, dtype is torch.float8_e4m3fn, ks, vs


def _span(t):
    """First and last address of a nonempty tensor's elements."""
    first, last = t.data_ptr(), -1
    for n, s in zip(t.shape, t.stride()):
        last += (n - 1) * s
    return first, first + (last + 2) * t.element_size() - 1


def _meet(a, b):
    return a[0] <= b[1] and b[0] <= a[1]


def _check_int32(device, name, t):
    if t is not None and (t.dtype is not torch.int32 or t.ndim != 1 or t.device != device or (t.stride(0) != 1 and t.numel() > 1)):
        raise ValueError(f'{name} must be contiguous int32 on the device of the pages')


def _check_table(device, table, lengths):
    """(sequences, pages per sequence, row stride) of a page table."""
    if table.ndim != 2 or table.dtype is not torch.int32 or table.device != device or not table.numel():
        raise ValueError('table must be int32 [sequences, pages per sequence] with contiguous rows, on the device of the pages')
    (sequences, width), strides = table.shape, table.stride()
    if strides[1] != 1:
        raise ValueError('table must be int32 [sequences, pages per sequence] with contiguous rows, on the device of the pages')
    _check_int32(device, 'lengths', lengths)
    if lengths.numel() != sequences:
        raise ValueError('lengths must hold one entry per row of table')
    return sequences, width, strides[0]


def _check_scales(device, hk, k_scale, v_scale, fp8):
    if k_scale is None and v_scale is None:
        return
    if not fp8:
        raise ValueError('scales come with float8_e4m3fn pages')
    for name, t in (('k_scale', k_scale), ('v_scale', v_scale)):
        if t is not None and (t.dtype is not torch.float32 or t.device != device or tuple(t.shape) != (hk,) or not t.is_contiguous()):
            raise ValueError(f'{name} must be contiguous float32 [kv_heads] on the device of the pages')


@lru_cache(maxsize=4096)
def _scratch_bytes(name, *sizes):
    return getattr(_lib.load(), name)(*sizes)


def paged_attention(q, k_pages, v_pages, table, lengths, *, slots=None, scale=None, k_scale=None, v_scale=None, return_lse=False, out=None):
    """Attention of one new token per sequence over a paged cache: q bf16 [batch, heads, dim], row b over the lengths[s] tokens of
    slot s = slots[b] (b by default), token t at k_pages[table[s, t // page], h // (heads / kv_heads), t % page].

    Pages [pages, kv_heads, page, dim] in bf16 or float8_e4m3fn (times k_scale / v_scale [kv_heads]), page a power of two, dim 64 or
    128; table int32 [sequences, pages per sequence], lengths int32 [sequences], slots int32 [batch], all read on the device:
    no host synchronisation. scale defaults to dim ** -0.5. Returns bf16 [batch, heads, dim], with return_lse also the float32
    natural log of each softmax's sum (-inf and zeros for an empty sequence). Sums are 32 bits wide; probabilities are
    rounded before they meet the values, by 2^-16 of themselves with bf16 pages, 2^-12 with E4M3 ones. Slots, lengths and table entries
    that lead outside are left out and reported by device_status(). Can be captured, except for a device's first paged call."""
    pages, hk, page, dim, fp8, ks, vs = _check_pages(k_pages, v_pages)
    dev = k_pages.device
    if q.ndim != 3 or q.dtype is not torch.bfloat16 or q.device != dev or q.shape[2] != dim or q.stride(2) != 1:
        raise ValueError('q must be BF16 [batch, heads, dim] with contiguous rows, on the device of the pages')
    shape = q.shape
    batch, hq, _ = shape
    if not batch or not hq or hq % hk:
        raise ValueError('a nonempty batch and a whole number of heads per kv head are required')
    sequences, width, table_stride = _check_table(dev, table, lengths)
    if slots is not None:
        _check_int32(dev, 'slots', slots)
    if (batch > sequences) if slots is None else (slots.numel() != batch):
        raise ValueError('slots must name one sequence per row of q')
    _check_scales(dev, hk, k_scale, v_scale, fp8)
    if q.requires_grad and torch.is_grad_enabled():
        raise RuntimeError('paged_attention is inference-only; use torch.inference_mode()')
    require_sm100(dev)
    qs = q.stride()
    if qs[0] % 2 or qs[1] % 2 or q.data_ptr() % 4:
        q = q.clone(memory_format=torch.contiguous_format)
        qs = q.stride()
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(shape)      # the former takes half the time of torch.empty
    elif out.shape != shape or out.dtype is not torch.bfloat16 or not out.is_contiguous() or out.device != dev:
        raise ValueError(f'out must be contiguous BF16 {tuple(shape)} on the device of the pages')
    elif _meet(_span(out), _span(q)):
        raise ValueError('out must not share memory with q')
    lse = q.new_empty((batch, hq), dtype=torch.float32) if return_lse else None
    lib = _lib.load()
    with _device(dev), _launching:
        stream = _stream(dev)
        scratch = _scratch(dev, stream, 'paged', _scratch_bytes('tw_paged_attention_workspace', batch, hq, hk, dim, width * page))
        args = _lib.PagedAttentionArgs(
            q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), table.data_ptr(), lengths.data_ptr(), None if slots is None else slots.data_ptr(),
            _ptr(k_scale), _ptr(v_scale), out.data_ptr(), None if lse is None else lse.data_ptr(), scratch.data_ptr(), _cache_status(dev), qs[0], qs[1],
            ks[0], ks[1], vs[0], vs[1], table_stride, dim ** -.5 if scale is None else scale, batch, sequences, hq, hk, dim, page, pages, width, fp8)
        _lib.check(lib.tw_paged_attention(ctypes.byref(args), stream))
    return (out, lse) if return_lse else out


def _cache(k_pages, v_pages, table, lengths, refs, page=None):
    """(argument struct, device, kv heads, dim, fp8, sequences) of a paged cache whose small tables are updated in place."""
    if k_pages is not None:
        pages, hk, page, dim, fp8, ks, vs = _check_pages(k_pages, v_pages)
        if (pages > 1 and not (ks[0] and vs[0])) or (hk > 1 and not (ks[1] and vs[1])):
            raise ValueError('pages are written: they must not be expanded')
        dev, pointers = k_pages.device, (k_pages.data_ptr(), v_pages.data_ptr())
        if pointers[0] == pointers[1]:
            raise ValueError('pages are written: k_pages and v_pages must not be the same memory')
    else:
        dev, pages, hk, dim, fp8, ks, vs, pointers = refs.device, refs.numel(), 0, 0, False, (0, 0), (0, 0), (None, None)
        if type(page) is not int or page < 1 or page & (page - 1):
            raise ValueError('tokens per page must be a power of two')
    sequences, width, table_stride = _check_table(dev, table, lengths)
    if sequences > 1 and table_stride < width:
        raise ValueError('table is written: its rows must not overlap')
    _check_int32(dev, 'refs', refs)
    if refs.numel() != pages:
        raise ValueError('refs must hold one count per page')
    require_sm100(dev)
    args = _lib.Cache(*pointers, table.data_ptr(), lengths.data_ptr(), refs.data_ptr(), _cache_status(dev), ks[0], ks[1], vs[0], vs[1], table_stride,
                      sequences, width, pages, hk, page, dim, fp8)
    return args, dev, hk, dim, fp8, sequences


def cache_append_(k, v, k_pages, v_pages, table, lengths, refs, *, slots=None, cu=None, k_scale=None, v_scale=None):
    """New tokens behind their sequences: rows k, v bf16 [rows, kv_heads, dim] go to the cache, row i behind the tokens of slot
    slots[i] (i by default), or with cu int32 [batch + 1] rows cu[i] ... cu[i + 1] - 1. New pages are the lowest free numbers, in the
    order of i; table, lengths and refs are updated. A slot may be named once. E4M3 pages hold k / k_scale[head] rounded, saturating.
    All on the device: a call that cannot be done (a full pool or table; a slot, length or partly filled last page outside) changes
    nothing and shows in device_status()."""
    args, dev, hk, dim, fp8, sequences = _cache(k_pages, v_pages, table, lengths, refs)
    shape = k.shape
    if len(shape) != 3 or shape != v.shape or shape[1] != hk or shape[2] != dim or k.dtype is not torch.bfloat16 or v.dtype is not torch.bfloat16 \
            or k.device != dev or v.device != dev:
        raise ValueError('k and v must be BF16 [rows, kv_heads, dim] alike, on the device of the pages')
    if (k.requires_grad or v.requires_grad) and torch.is_grad_enabled():
        raise RuntimeError('the cache is inference-only; use torch.inference_mode()')
    _check_int32(dev, 'slots', slots)
    _check_int32(dev, 'cu', cu)
    _check_scales(dev, hk, k_scale, v_scale, fp8)
    rows = shape[0]
    batch = slots.numel() if slots is not None else (cu.numel() - 1 if cu is not None else rows)
    if (cu is None and batch != rows) or (cu is not None and (cu.numel() != batch + 1 or batch < 0)):
        raise ValueError('one row per slot, or cu with one offset more than there are slots, is required')
    if slots is None and batch > sequences:
        raise ValueError('more entries than sequences')
    if batch < 1 or not rows:
        return
    ks, vs = k.stride(), v.stride()
    if ks[2] != 1 or ks[0] % 8 or ks[1] % 8 or k.data_ptr() % 16:
        k = k.clone(memory_format=torch.contiguous_format)
        ks = k.stride()
    if vs[2] != 1 or vs[0] % 8 or vs[1] % 8 or v.data_ptr() % 16:
        v = v.clone(memory_format=torch.contiguous_format)
        vs = v.stride()
    pages, _, page, _ = k_pages.shape
    width = 1 if fp8 else 2
    k_at, v_at, new_k, new_v = args.k_pages, args.v_pages, k.data_ptr(), v.data_ptr()
    k_end = k_at + ((pages - 1) * args.k_stride_page + (hk - 1) * args.k_stride_head + page * dim) * width
    v_end = v_at + ((pages - 1) * args.v_stride_page + (hk - 1) * args.v_stride_head + page * dim) * width
    for at, (row, head, _) in ((new_k, ks), (new_v, vs)):
        end = at + ((rows - 1) * row + (hk - 1) * head + dim) * 2
        if (at < k_end and k_at < end) or (at < v_end and v_at < end):
            raise ValueError('k and v must not lie in the pages')
    call = _lib.AppendArgs(new_k, new_v, _ptr(slots), _ptr(cu), _ptr(k_scale), _ptr(v_scale), ks[0], ks[1], vs[0], vs[1], batch, rows)
    with _device(dev), _launching:
        stream = _stream(dev)
        scratch = _scratch(dev, stream, 'paged', _scratch_bytes('tw_cache_append_workspace', batch, rows))
        _lib.check(_lib.load().tw_cache_append(ctypes.byref(args), ctypes.byref(call), scratch.data_ptr(), stream))


def cache_fork_(k_pages, v_pages, table, lengths, refs, parents, children):
    """Slot children[i], which must be empty and may be named once, becomes a copy of slot parents[i] as it was before the call: full
    pages are shared (refs counts their holders), the rows of a partly filled last page are copied to the lowest free page. int32 [n]
    each. A call that cannot be done (a full pool; a slot, length or page of a parent outside) changes nothing and shows in
    device_status()."""
    args, dev, *_ = _cache(k_pages, v_pages, table, lengths, refs)
    _check_int32(dev, 'parents', parents)
    _check_int32(dev, 'children', children)
    count = parents.numel()
    if children.numel() != count:
        raise ValueError('one child per parent is required')
    if not count:
        return
    with _device(dev), _launching:
        stream = _stream(dev)
        scratch = _scratch(dev, stream, 'paged', _scratch_bytes('tw_cache_fork_workspace', count))
        _lib.check(_lib.load().tw_cache_fork(ctypes.byref(args), parents.data_ptr(), children.data_ptr(), count, scratch.data_ptr(), stream))


def cache_free_(table, lengths, refs, slots, page_size):
    """Empties slots int32 [n] of a cache with page_size tokens per page: their pages lose a reference, their table entries become -1. A
    slot named twice is freed once; one outside is left out and shows in device_status()."""
    args, dev, *_ = _cache(None, None, table, lengths, refs, page_size)
    _check_int32(dev, 'slots', slots)
    if slots.numel():
        with _device(dev):
            _lib.check(_lib.load().tw_cache_free(ctypes.byref(args), slots.data_ptr(), slots.numel(), _stream(dev)))


def cache_compact_(k_pages, v_pages, table, lengths, refs):
    """Moves the live pages to the numbers 0 ... live - 1 (the r-th live page at or above live to the r-th free one below), updates table
    and refs, and returns live as an int32 scalar tensor. A table entry outside the pool stays as it is and shows in device_status()."""
    args, dev, *_ = _cache(k_pages, v_pages, table, lengths, refs)
    live = torch.empty((), device=dev, dtype=torch.int32)
    with _device(dev), _launching:
        stream = _stream(dev)
        scratch = _scratch(dev, stream, 'paged', _scratch_bytes('tw_cache_compact_workspace', refs.numel()))
        _lib.check(_lib.load().tw_cache_compact(ctypes.byref(args), live.data_ptr(), scratch.data_ptr(), stream))
    return live


STATUS_KEYS = {'g': 0, 'a': 0, 'q': 8, 'c': 0}   # workspace -> byte offset of its device status word: fused GEMM, attention, quantizer, paged cache


def device_status(device=None):
    """Worst status word any kernel of this device wrote on a bounded-wait timeout (0 = none); waits for all streams of the device,
    so not while one of them is being captured.
    Covers the fused GEMM, the attention kernel and the single-pass quantizer's grid barrier: each writes into its own workspace;
    and what the operators of the paged cache found and left out (an entry outside the cache, a full pool)."""
    dev = torch.device('cuda', torch.cuda.current_device()) if device is None else torch.device(device)
    if dev.index is None:
        dev = torch.device('cuda', torch.cuda.current_device())
    torch.cuda.synchronize(dev)
    worst = 0
    for key, offset in STATUS_KEYS.items():
        ws = _workspaces.get((dev, key))
        if ws is not None:
            worst = max(worst, int(ws[offset:offset + 4].view(torch.int32).item()))
    return worst


def reset_device_status(device=None):
    """Clear the status words (after a reported timeout has been handled); waits for all streams of the device, before and after."""
    dev = torch.device('cuda', torch.cuda.current_device()) if device is None else torch.device(device)
    if dev.index is None:
        dev = torch.device('cuda', torch.cuda.current_device())
    torch.cuda.synchronize(dev)
    for key, offset in STATUS_KEYS.items():
        ws = _workspaces.get((dev, key))
        if ws is not None:
            ws[offset:offset + 4].zero_()
    torch.cuda.synchronize(dev)


# ---- pointwise producers with fused tensor factor -----------------------------------------------
# Host mirrors of activate_with_factor (thunderworld_fp4/_fusion.py:26-34) and nemotron_norm
# (thunderworld_fp4/cosmos/norm_fusion.py:29-43); same argument checks and error types.
ACT_MODES = {'relu2': 0, 'mul': 1, 'gelu_tanh': 2}


def _check_bf16(*tensors):
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda or t.dtype != torch.bfloat16 or not t.is_contiguous():
            raise ValueError('expected contiguous CUDA BF16 tensors')


def _stats(device, want):
    """(stats[2] float32, scratch) or (None, None). The scratch is the stream's, or the capture's: a maximum and a ticket that calls
    on two streams must not share."""
    if not want:
        return None, None
    return torch.empty(2, device=device, dtype=torch.float32), _scratch(device, _stream(device))


def activate_with_factor(a, b=None, *, mode=None, want_factor=True, return_stats=False):
    """y = relu(a)^2 (b None), a * b, or gelu_tanh(a) (mode='gelu_tanh'); returns (y, factor) with
    factor = max|y| / 2688 as a 0-d float32 tensor (or None); return_stats: the pair (factor, max|y|) instead."""
    if torch.is_grad_enabled() and (a.requires_grad or (b is not None and b.requires_grad)):
        raise RuntimeError('fused activations are inference only')
    _check_bf16(a, b)
    if b is not None and b.shape != a.shape:
        raise ValueError('operands must have equal shapes')
    require_sm100(a.device)
    mode = ACT_MODES[mode or ('relu2' if b is None else 'mul')]
    y = torch.empty_like(a)
    stats, scratch = _stats(a.device, want_factor)
    _lib.check(_lib.load().tw_activate(_ptr(a), _ptr(b), _ptr(y), _ptr(stats), _ptr(scratch), a.numel(), mode, _stream(a.device)))
    return y, (None if stats is None else (stats if return_stats else stats[0]))


def rms_norm(x, weight=None, eps=1e-6, *, shift=None, scale=None, want_factor=False, return_stats=False):
    """RMSNorm over the last dimension, optional weight, optional AdaLN modulation with shift/scale of shape
    [batch, hidden] (x is [batch, tokens, hidden]). Returns y or (y, factor); return_stats: (y, (factor, max|y|))."""
    if torch.is_grad_enabled() and x.requires_grad:
        raise RuntimeError('Fused RMSNorm requires inference mode')
    _check_bf16(x, weight, shift, scale)
    hidden = x.shape[-1]
    if weight is not None and weight.numel() != hidden:
        raise ValueError('Fused RMSNorm supports BF16 inputs matching the weight')
    if (shift is None) != (scale is None):
        raise ValueError('shift and scale come together')
    rows = x.numel() // hidden
    per_batch = rows
    if shift is not None:
        if shift.shape != scale.shape or shift.shape[-1] != hidden or rows % (shift.numel() // hidden):
            raise ValueError('shift/scale must be [batch, hidden] with batch dividing the rows of x')
        per_batch = rows // (shift.numel() // hidden)
    require_sm100(x.device)
    y = torch.empty_like(x)
    stats, scratch = _stats(x.device, want_factor)
    _lib.check(_lib.load().tw_rms_norm(_ptr(x), _ptr(weight), _ptr(shift), _ptr(scale), _ptr(y), _ptr(stats), _ptr(scratch),
                                       rows, hidden, per_batch, float(eps), _stream(x.device)))
    if not want_factor:
        return y
    return (y, stats) if return_stats else (y, stats[0])


def rms_norm_heads(x, eps=1e-6):
    """RMSNorm over head_dim = 128 of a (possibly strided) view [..., tokens, heads, 128] whose leading
    dimensions fold into the token stride; returns a contiguous tensor of the same shape."""
    if x.dtype != torch.bfloat16 or not x.is_cuda or x.shape[-1] != 128 or x.stride(-1) != 1:
        raise ValueError('expected a CUDA BF16 view [..., heads, 128] with unit inner stride')
    require_sm100(x.device)
    heads = x.shape[-2]
    lead = x.reshape(-1, heads, 128) if x.dim() != 3 else x       # a view when the leading dims are foldable
    if lead.data_ptr() != x.data_ptr():
        raise ValueError('leading dimensions must fold into one token stride')
    y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    _lib.check(_lib.load().tw_rms_norm_heads(_ptr(lead), _ptr(y), lead.shape[0], heads, lead.stride(0), lead.stride(1),
                                             float(eps), _stream(x.device)))
    return y


def rope_heads(x, cos, sin, *, norm=False, eps=1e-6):
    """Rotary embedding of a (possibly strided) bf16 view [..., tokens, heads, 128] with the reference's rounding
    sequence (fused_rope, thunderworld_fp4/cosmos/pipeline_tuning.py:57-63); cos / sin [table_rows, 128], float32 or
    bf16, row token % table_rows. norm=True runs the head RMSNorm first in the same pass. Returns a contiguous tensor."""
    if x.dtype != torch.bfloat16 or not x.is_cuda or x.shape[-1] != 128 or x.stride(-1) != 1:
        raise ValueError('expected a CUDA BF16 view [..., heads, 128] with unit inner stride')
    if cos.shape != sin.shape or cos.ndim != 2 or cos.shape[1] != 128 or cos.dtype != sin.dtype or \
            cos.dtype not in (torch.float32, torch.bfloat16) or not cos.is_contiguous() or not sin.is_contiguous():
        raise ValueError('cos / sin must be contiguous [rows, 128] tables of one dtype (float32 or bfloat16)')
    require_sm100(x.device)
    heads = x.shape[-2]
    lead = x.reshape(-1, heads, 128) if x.dim() != 3 else x
    if lead.data_ptr() != x.data_ptr():
        raise ValueError('leading dimensions must fold into one token stride')
    y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    _lib.check(_lib.load().tw_rope_heads(_ptr(lead), _ptr(y), lead.shape[0], heads, lead.stride(0), lead.stride(1), _ptr(cos),
                                         _ptr(sin), cos.shape[0], int(cos.dtype == torch.bfloat16), int(norm), float(eps),
                                         _stream(x.device)))
    return y


def _overlap(a, b):
    """Whether two contiguous tensors share memory."""
    return a.data_ptr() < b.data_ptr() + b.numel() * b.element_size() and b.data_ptr() < a.data_ptr() + a.numel() * a.element_size()


def gate_residual_norm_(x, y, gate=None, *, post_norm=False, post_weight=None, residual_scale=1., weight=None, shift=None,
                        scale=None, eps=1e-6, want_factor=False, return_stats=False):
    """The gated residual and the norm that follows it in one pass: x = residual_scale * x + gate[:, None, :] * z in place,
    where z is y, or with post_norm (implied by post_weight) the RMSNorm of y times post_weight; returns
    rms_norm(x, weight, eps, shift=shift, scale=scale, ...) of the new x, with want_factor / return_stats as there.
    x, y [batch, tokens, hidden]; gate, shift, scale [batch, hidden]; gate None: ones. Without post_norm and with
    residual_scale 1 the bits are those of gate_residual_ followed by rms_norm."""
    dev, hidden, size = x.device, x.shape[-1], x.numel()
    grad = torch.is_grad_enabled()
    for t in (x, y, gate, post_weight, weight, shift, scale):
        if t is not None:
            if grad and t.requires_grad:
                raise RuntimeError('Fused residual and norm requires inference mode')
            if t.dtype is not torch.bfloat16 or not t.is_cuda or not t.is_contiguous():
                raise ValueError('expected contiguous CUDA BF16 tensors')
            if t.device != dev:
                raise ValueError('all operands must be on one device')
    if y.shape != x.shape:
        raise ValueError('x and y must have equal shapes')
    if not size:
        raise ValueError('empty residual streams are unsupported')
    for t in (weight, post_weight):
        if t is not None and t.numel() != hidden:
            raise ValueError('norm weights must be [hidden]')
    if (shift is None) != (scale is None):
        raise ValueError('shift and scale come together')
    rows = per_batch = size // hidden
    lead = gate if gate is not None else shift
    if lead is not None:
        batch = lead.numel() // hidden
        for t in (gate, shift, scale):
            if t is not None and (t.shape[-1] != hidden or t.numel() != batch * hidden):
                raise ValueError('gate, shift and scale must be [batch, hidden]')
        if not batch or rows % batch:
            raise ValueError('gate, shift and scale must be [batch, hidden] with batch dividing the rows of x')
        per_batch = rows // batch
    if _overlap(x, y):
        raise ValueError('x is updated in place and must not share memory with y')
    require_sm100(dev)
    h = torch.empty_like(x)
    stats = torch.empty(2, device=dev, dtype=torch.float32) if want_factor else None
    with _device(dev):
        stream = _stream(dev)
        _lib.check(_lib.load().tw_gate_residual_norm(
            _ptr(x), _ptr(y), _ptr(gate), _ptr(post_weight), int(post_norm or post_weight is not None), float(residual_scale),
            _ptr(weight), _ptr(shift), _ptr(scale), _ptr(h), _ptr(stats), _ptr(_scratch(dev, stream)) if want_factor else None,
            rows, hidden, per_batch, float(eps), stream))
    if not want_factor:
        return h
    return (h, stats) if return_stats else (h, stats[0])


def gate_residual_(x, gate, y):
    """x += gate[:, None, :] * y in place; x, y [batch, tokens, hidden], gate [batch, hidden]."""
    _check_bf16(x, gate, y)
    hidden = x.shape[-1]
    rows = x.numel() // hidden
    if y.shape != x.shape or gate.shape[-1] != hidden or rows % (gate.numel() // hidden):
        raise ValueError('shapes do not match')
    require_sm100(x.device)
    _lib.check(_lib.load().tw_gate_residual(_ptr(x), _ptr(gate), _ptr(y), rows, hidden, rows // (gate.numel() // hidden),
                                            _stream(x.device)))
    return x
