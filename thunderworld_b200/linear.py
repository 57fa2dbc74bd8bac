"""W4A4 (+A1·W4) linear over immutable packed NVFP4 weights: the reference's `FP4Linear` and `_pack`
(packages/fp4-repair/src/thunderworld_fp4/linear.py:13-135) on the sm_100a kernels.

Packed format: low nibble first, uint8 [N,K/2]; un-swizzled E4M3 [N,K/16]; scalar weight global scale;
weight = decoded codes * scale * global scale. Forward rounds (x * prescale) to BF16 before activation
quantization. N and K are multiples of 128; explicit masks index M128/N128/K128 tiles.
"""
import torch
from . import ops
from .config import LinearRepairConfig


def _pack(x, prescale, repair, full, union, **kw):
    """Activation packer with the reference's signature: returns (codes, scales, factor, mp) as a
    `Packed` (which unpacks like that tuple and also carries the atom-layout scales)."""
    mode = 0 if not repair else (1 if full else 2)
    return ops.quantize(x, prescale, repair=mode, mask=union if mode == 2 else None, **kw)


def sampled_block_rank(x, prescale, m, k):
    """Rank of every K128 block within its M128 row block by sampled energy: eight rows and eight
    columns (every 16th) of bf16(x*d) per 128x128 block, rank 0 = largest, lower index wins ties
    (reference: activation_rank, _linear_kernels.py:23-34). One CUDA launch; no host sync."""
    return ops.activation_rank(x, prescale)


class FP4Linear(torch.nn.Module):
    """W4A4(+A1W4) for FFN or projection layers, with independent configuration."""

    def __init__(self, weight_codes, weight_scales, weight_global_scale, *, prescale=None, bias=None, config=None):
        super().__init__()
        if weight_codes.ndim != 2 or weight_codes.dtype != torch.uint8:
            raise ValueError('weight_codes must be uint8 [N,K/2]')
        n, half = weight_codes.shape
        self.in_features, self.out_features = half * 2, n
        config = config or LinearRepairConfig()
        if not isinstance(config, LinearRepairConfig):
            raise TypeError('config must be LinearRepairConfig')
        counts = config.output_counts(n, half * 2)
        if weight_scales.shape != (n, half * 2 // 16) or weight_scales.dtype != torch.float8_e4m3fn:
            raise ValueError('weight_scales must be un-swizzled E4M3 [N,K/16]')
        device = weight_codes.device
        if weight_scales.device != device:
            raise ValueError('weight codes/scales must be on the same device')
        factor = torch.as_tensor(weight_global_scale, device=device, dtype=torch.float32)
        if factor.numel() != 1 or not bool(torch.isfinite(factor).all()) or not bool((factor > 0).all()):
            raise ValueError('weight_global_scale must be one finite positive value')
        if not bool(torch.isfinite(weight_scales.float()).all()) or bool((weight_scales.float() < 0).any()):
            raise ValueError('weight scales must be finite and nonnegative')
        if prescale is None:
            prescale = torch.ones(self.in_features, device=device, dtype=torch.float32)
        if prescale.shape != (self.in_features,) or not bool(torch.isfinite(prescale).all()) or not bool((prescale > 0).all()):
            raise ValueError('prescale must be a finite positive [K] vector')
        if bias is not None and (bias.shape != (n,) or not bool(torch.isfinite(bias).all())):
            raise ValueError('bias must be a finite [N] vector')
        self.register_buffer('weight_codes', weight_codes.detach().contiguous().clone())
        self.register_buffer('weight_scales', weight_scales.detach().contiguous().clone())
        self.register_buffer('weight_global_scale', factor.reshape(()).detach().clone())
        self.register_buffer('prescale', prescale.detach().to(device=device, dtype=torch.float32).contiguous())
        self.register_buffer('bias', None if bias is None else bias.detach().to(device=device, dtype=torch.bfloat16).contiguous())
        self._config = config
        kb = self.in_features // 128
        self._repair, self._full = any(counts), all(c == kb for c in counts)
        self.register_buffer('_counts', torch.tensor(counts, device=device, dtype=torch.int32), persistent=False)
        self._scales_swz = None

    @property
    def config(self):
        """Immutable configuration; construct another module to change quotas."""
        return self._config

    @classmethod
    @torch.no_grad()
    def from_float(cls, weight, *, prescale=None, bias=None, config=None):
        """Offline round-to-nearest W4 preparation of W / prescale (not a calibration)."""
        if weight.ndim != 2 or not weight.is_cuda or weight.dtype != torch.bfloat16:
            raise ValueError('offline weight must be BF16 CUDA [N,K]')
        ops.require_sm100(weight.device)
        n, k = weight.shape
        (config or LinearRepairConfig()).output_counts(n, k)
        d = torch.ones(k, device=weight.device) if prescale is None else prescale.to(weight.device).float()
        if d.shape != (k,) or not bool(torch.isfinite(d).all()) or not bool((d > 0).all()):
            raise ValueError('prescale must be positive finite [K]')
        transformed = (weight.float() / d).bfloat16().contiguous()
        packed = _pack(transformed, None, False, False, None)
        return cls(packed.codes[0, :n], packed.scales[0, :n], packed.factor, prescale=d, bias=bias, config=config)

    def forward(self, x, *, repair_mask=None):
        if x.ndim < 2 or x.shape[-1] != self.in_features or x.dtype != torch.bfloat16:
            raise ValueError('expected BF16 input [..., K]')
        if not x.is_cuda or x.device != self.weight_codes.device:
            raise ValueError('activation and packed weights must share a CUDA device')
        ops.require_sm100(x.device)
        if torch.is_grad_enabled() and x.requires_grad:
            raise RuntimeError('FP4Linear is inference-only; use torch.inference_mode()')
        flat = x.reshape(-1, self.in_features).contiguous()
        m, k, n = flat.shape[0], self.in_features, self.out_features
        if m == 0:
            raise ValueError('empty activation rows are unsupported')
        shape = (ops.cdiv(m, 128), n // 128, k // 128)
        mask = None
        if repair_mask is not None:
            if (repair_mask.shape != shape or repair_mask.dtype != torch.bool or repair_mask.device != x.device
                    or not repair_mask.is_contiguous()):
                raise ValueError(f'repair_mask must be contiguous CUDA bool {shape}')
            mask, repair, full = repair_mask, True, False
        elif self._repair and not self._full:
            ranks = sampled_block_rank(flat, self.prescale, m, k)
            mask = (ranks[:, None, :] < self._counts[None, :, None]).contiguous()
            repair, full = True, False
        else:
            repair, full = self._repair, self._full
        union = mask.any(dim=1).contiguous() if mask is not None else None
        if self._scales_swz is None:
            self._scales_swz = ops.swizzle(self.weight_scales)
        packed = _pack(flat, self.prescale, repair, full, union, wg=self.weight_global_scale)
        na = 0 if not repair else (k // 128 if full else 1)
        out = ops.fused_gemm(m, n, k, packed, self.weight_codes, self._scales_swz, packed.alpha, na=na, mask=mask,
                             ws=self.weight_scales, mask_per_n=mask is not None, bias=self.bias)
        return out.reshape(*x.shape[:-1], n)

    def matvec(self, x, *, out_dtype=torch.bfloat16):
        """The layer for a token at a time: at most 32 rows [..., K], which stay BF16 (no activation planes, hence nothing to
        repair); the same weights, prescale and bias as forward()."""
        return ops.fp4_matvec(x, self.weight_codes, self.weight_scales, self.weight_global_scale, prescale=self.prescale,
                              bias=self.bias, out_dtype=out_dtype)
