"""Rotary position embedding on the GPU.

``rotary`` is the drop-in for the reference's exact bf16 BSND rotary
(qwen3_tts_engine/rotary_triton_ascend.py:29-44): same arguments, same validation, a new
output tensor, and torch-eager rounding after every op (kernel ``q3t_rotary``); fp32 rows
are accepted too, with torch-eager fp32 rounding.
``rope_tables`` produces the default-RoPE cos/sin rows for integer positions
(kernel ``q3t_rope_tables``); ``inverse_frequencies`` is the host-side fp32 table it uses.
``rotary_axes`` rotates queries and keys of tokens with a position on each of several axes (the
talker's ``mrope_section``; time, height and width of images and video; kernel
``q3t_rotary_axes``).
"""
import math

import torch

from . import _lib

DEFAULT_THETA = 1_000_000.0
_INV_FREQ = {}


def rotary(hidden, cos, sin):
    """Rotate-half RoPE of a contiguous bf16 (batch, length, heads, width) tensor."""
    if hidden.ndim != 4 or hidden.device.type != 'cuda' or hidden.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError('Expected BF16 or FP32 BSND ROCm input')
    batch, length, heads, width = hidden.shape
    if heads < 1 or width not in (64, 128) or batch * length < 1:
        raise ValueError('Unsupported rotary shape')
    if cos.shape != (batch, length, width) or sin.shape != cos.shape:
        raise ValueError('Rotary coefficients must match batch, length and width')
    if any(t.device != hidden.device or t.dtype != hidden.dtype or not t.is_contiguous()
           for t in (hidden, cos, sin)):
        raise ValueError('Rotary tensors must be contiguous with matching dtype/device')
    output = torch.empty_like(hidden)
    status = _lib.library().q3t_rotary(hidden.data_ptr(), cos.data_ptr(), sin.data_ptr(),
                                       output.data_ptr(), batch * length, heads, width,
                                       _lib.DTYPE_CODES[hidden.dtype],
                                       _lib.stream_handle(hidden.device))
    _lib.check(status, 'rotary')
    return output


def inverse_frequencies(head_dim, theta=DEFAULT_THETA):
    """fp32 1 / theta**(2i/head_dim), computed as the default RoPE initialiser does."""
    exponent = torch.arange(0, head_dim, 2, dtype=torch.int64).to(torch.float32) / head_dim
    return 1.0 / (theta ** exponent)


def rope_tables(positions, head_dim, theta=DEFAULT_THETA, scaling=1.0, dtype=torch.bfloat16,
                inv_freq=None):
    """cos, sin of shape positions.shape + (head_dim,) for int64 device positions."""
    if positions.dtype != torch.int64 or positions.device.type != 'cuda':
        raise ValueError('positions must be an int64 ROCm tensor')
    if dtype not in (torch.bfloat16, torch.float32):
        raise ValueError('rope tables are produced in bf16 or fp32')
    if head_dim % 2 or head_dim < 2:
        raise ValueError('head_dim must be even')
    if inv_freq is None:
        key = (positions.device, head_dim, float(theta))
        inv_freq = _INV_FREQ.get(key)
        if inv_freq is None:  # cached so that captured graphs never see a host copy
            inv_freq = inverse_frequencies(head_dim, theta).to(positions.device)
            _INV_FREQ[key] = inv_freq
    inv_freq = inv_freq.to(device=positions.device, dtype=torch.float32).contiguous()
    flat = positions.contiguous().view(-1)
    cos = torch.empty(*positions.shape, head_dim, device=positions.device, dtype=dtype)
    sin = torch.empty_like(cos)
    status = _lib.library().q3t_rope_tables(flat.data_ptr(), flat.numel(), inv_freq.data_ptr(),
                                            head_dim // 2, float(scaling),
                                            _lib.DTYPE_CODES[dtype], cos.data_ptr(),
                                            sin.data_ptr(), _lib.stream_handle(positions.device))
    _lib.check(status, 'rope tables')
    return cos, sin


_pack_axes = _lib.packer(_lib.RotaryAxesArgs)
_ROTARY_TYPES = {torch.bfloat16: _lib.Q3T_BF16, torch.float16: _lib.Q3T_F16, torch.float32: _lib.Q3T_F32}
_TURNS = {}


def _turns(half, theta, like):
    """Full turns per position of every frequency, theta**(-i/half) / 2 pi, in float64."""
    theta = float(theta)
    key = (like.get_device(), half, theta)
    turns = _TURNS.get(key)
    if turns is None:
        if not 0 < theta < math.inf:
            raise ValueError('theta must be positive')
        # kept, but a graph being captured forms its own: it takes no host copy, and its memory is its own
        with torch.cuda.device(like.device):
            capturing = torch.cuda.is_current_stream_capturing()
        exponent = torch.arange(half, dtype=torch.float64, device=like.device if capturing else None) / half
        turns = (theta ** -exponent / (2 * math.pi)).to(like.device)
        if not capturing:
            _TURNS[key] = turns
    return turns


def _dims(t):
    """(stride, size) of the dimensions of rows t that have more than one entry, outermost first."""
    return sorted(((s, n) for n, s in zip(t.shape[:-1], t.stride()) if n > 1), reverse=True)


def _extent(dims, row):
    """Elements from the first to the last of rows of ``row`` elements."""
    return sum((n - 1) * s for s, n in dims) + row


def _share_memory(x, y=None):
    """Whether rows of x overlap each other, or rows of y; True as well where no nesting of the
    dimensions (each stride passes all that lies within it) shows that they do not."""
    if x.numel() == 0 or (y is not None and y.numel() == 0):
        return False
    row, dims = x.shape[-1], _dims(x)
    if y is None:
        return any(s < _extent(dims[i + 1:], row) for i, (s, _) in enumerate(dims))
    others, apart = _dims(y), (y.data_ptr() - x.data_ptr()) // x.element_size()
    while True:
        ends = _extent(dims, row), apart + _extent(others, row)
        if apart >= ends[0] or ends[1] <= 0:
            return False
        if not dims or not others or dims[0][0] != others[0][0]:
            return True
        dims, others, stride = dims[1:], others[1:], dims[0][0]
        if max(_extent(dims, row), apart + _extent(others, row)) - min(0, apart) > stride:
            return True


def rotary_axes(query, key, positions, sections, *, interleaved=False, theta=DEFAULT_THETA, inv_freq=None,
                scaling=1.0, inplace=False):
    """Rotate-half RoPE of tokens that have a position on each of several axes.

    query (B, S, Hq, D) and key (B, S, Hkv, D), or None: bf16, fp16 or fp32 rows of any strides
    with unit-stride elements (views of the fused QKV projection are fine); positions (A, B, S)
    int64, A in 1 ... 4.  ``sections`` are the axes' shares of the ``half = sum(sections)``
    frequencies theta**(-i/half), or of ``inv_freq`` (half,), consecutively, or ``interleaved``:
    frequency i then belongs to axis ``a = i % A`` where ``i < A * sections[a]``, else to axis 0
    (the talker's ``mrope_section`` with ``interleaved``).  Elements i and i + half turn by
    ``positions[axis(i)] * frequency_i``; elements past ``2 * half`` are copied; cos and sin are
    multiplied by ``scaling``.  Angles are formed in float64, the rest in float32, and each element
    is rounded once (``rotary``, given cos/sin rows, rounds as torch-eager does).

    Returns (query, key) rotated: new contiguous tensors, or with ``inplace`` the given ones,
    rotated where they are (their rows must not overlap).  Inference only, as ``rotary``."""
    if query.ndim != 4 or (key is not None and key.ndim != 4):
        raise ValueError('expected BSND query and key rows')
    batch, tokens, q_heads, width = query.shape
    dtype = query.dtype
    if dtype not in _ROTARY_TYPES or (key is not None and key.dtype != dtype):
        raise ValueError('rotary supports bf16, fp16 or fp32 tensors of one dtype')
    half, axes = 0, len(sections)
    for n in sections:
        if not isinstance(n, int) or n < 0:
            raise ValueError('sections must be counts of frequencies')
        half += n
    if not 1 <= axes <= 4 or half < 1 or 2 * half > width or half > 512:
        raise ValueError('one to four sections must sum to at least one and at most half of the width (512 at most)')
    if positions.dtype != torch.int64 or positions.shape != (axes, batch, tokens):
        raise ValueError('positions must be an int64 (axes, batch, length) tensor')
    qs, ps, ks, k_heads = query.stride(), positions.stride(), (0, 0, 0, 1), 0
    if key is None:
        device = _lib.gpu_index(query, positions)
    else:
        key_batch, key_tokens, k_heads, key_width = key.shape
        if key_batch != batch or key_tokens != tokens or key_width != width:
            raise ValueError('query and key rows must have one batch, length and width')
        ks = key.stride()
        device = _lib.gpu_index(query, key, positions)
    if qs[3] != 1 or ks[3] != 1 or q_heads < 1 or (key is not None and k_heads < 1):
        raise ValueError('rows must be unit-stride, at least one per token')
    if inv_freq is None:
        turns = _turns(half, theta, query)
    else:
        if inv_freq.shape != (half,):
            raise ValueError('inv_freq must have one entry per frequency')
        turns = (inv_freq.to(device=query.device, dtype=torch.float64) / (2 * math.pi)).contiguous()
    if inplace:
        if _share_memory(query) or (key is not None and (_share_memory(key) or _share_memory(query, key))):
            raise ValueError('rows that share memory cannot be rotated in place')
        q_out, k_out, qos, kos = query, key, qs, ks
    else:
        q_out, k_out, kos = torch.empty_like(query, memory_format=torch.contiguous_format), None, (0, 0, 0)
        qos = (tokens * q_heads * width, q_heads * width, width)
        if key is not None:
            k_out = torch.empty_like(key, memory_format=torch.contiguous_format)
            kos = (tokens * k_heads * width, k_heads * width, width)
    if batch == 0 or tokens == 0:
        return q_out, k_out
    _lib.launch('q3t_rotary_axes', _pack_axes(
        batch, tokens, q_heads, k_heads, width, _ROTARY_TYPES[dtype], axes, *sections, *(0,) * (4 - axes), bool(interleaved),
        scaling, turns.data_ptr(), positions.data_ptr(), ps[0], ps[1], ps[2],
        query.data_ptr(), 0 if key is None else key.data_ptr(), qs[0], qs[1], qs[2], ks[0], ks[1], ks[2],
        q_out.data_ptr(), 0 if key is None else k_out.data_ptr(), qos[0], qos[1], qos[2], kos[0], kos[1], kos[2]),
        device, 'rotary axes')
    return q_out, k_out
