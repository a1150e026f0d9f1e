"""Operators on a paged key/value cache: what stands between the delta layers of a decode step.

  rotary            queries and keys turned to their positions
  append_kv         the same for the tokens of a step, their keys and values stored in the cache
  paged_attention   one new token per row over the pages of its table
  copy_pages        pages copied within every pool (forks, compaction)

They stand where the reference's serving engine has its own kernels for these (serving/csrc/pos_encoding,
serving/csrc/cache_kernels, serving/csrc/attention) and take the place of plain tensor operations over a padded
cache.  float16 and bfloat16; arithmetic in 32 bits and more, one rounding per output.  Work is enqueued on the
current stream of the tensors' device; nothing synchronises, and everything can be captured into a graph.  They serve
inference: no gradients are recorded.

What only the kernels can see -- a page or slot outside the pool, a length beyond the table -- goes to a status word that
`ops.poll_status` (`DeltaModelManager.check_status`) looks at with the others: `ops.DeltaKernelError`.
"""
from __future__ import annotations

import ctypes as C
import math
import struct
from functools import lru_cache
from typing import Dict, Mapping, NamedTuple, Optional, Sequence, Tuple, Union

import numpy as np
import torch

from . import _lib, ops

_TYPES = {torch.float16: 0, torch.bfloat16: 1}
_ATTENTION = struct.Struct("=q9Q2q11q8ifi")       # dz_attention_args
_ROTARY = struct.Struct("=q10Qq14q8ifi")          # dz_rotary_args
MAX_DIM = 256
COUNTERS = 32768                  # DZ_ATTENTION_COUNTERS


class RotaryPositions:
    """The angles of rotary positions: the first `rotary_dim` values of a head (default: all) are turned in
    pairs -- (i, i + rotary_dim / 2), or neighbours with `interleaved` -- by position * base^(-2 i / rotary_dim).

    `scaling` is the entry of a model's configuration that stretches the positions beyond the trained ones
    (`max_position`), as the reference's model layers read it (serving/vllm/model_executor):
      {"type": "linear", "factor": s}    positions divided by s
      {"type": "dynamic", "factor": s}   the base raised for s times the trained length
      {"type": "yarn", "factor": s, "original_max_position_embeddings": m, "extrapolation_factor": 1, "attn_factor": 1,
       "beta_fast": 32, "beta_slow": 1}  pairs that turn less than beta_slow times within m positions stretched, those that turn
                                         more than beta_fast kept, a ramp between; turned values times attn_factor (0.1 ln s + 1)
    Angles are held in 64 bits, as turns per position, on the host: a call takes them along."""

    def __init__(self, head_dim: int, rotary_dim: Optional[int] = None, base: float = 10000.0, max_position: int = 4096,
                 interleaved: bool = False, scaling: Optional[Mapping] = None) -> None:
        r = head_dim if rotary_dim is None else rotary_dim
        if head_dim < 2 or head_dim > MAX_DIM or head_dim % 2:
            raise ValueError(f"head_dim must be even, up to {MAX_DIM}")
        if r < 2 or r > head_dim or r % 2:
            raise ValueError("rotary_dim must be even and at most head_dim")
        if not base > 1 or max_position < 1:
            raise ValueError("base must be above 1 and max_position positive")
        self.head_dim, self.rotary_dim, self.interleaved = head_dim, r, bool(interleaved)
        self.attention_factor = 1.0
        kind, s = None, 1.0
        if scaling:
            scaling = dict(scaling)
            kind, s = scaling.pop("type", scaling.pop("rope_type", None)), scaling.pop("factor", None)
            if kind is None:
                raise ValueError("a scaling must name its type")
            if kind not in ("linear", "dynamic", "yarn"):
                raise NotImplementedError(f"positions scaled by {kind!r}: linear, dynamic and yarn are known")
            if s is None or not 1.0 <= float(s) < math.inf:
                raise ValueError("a scaling must have a factor of at least 1")
            s = float(s)
        i = np.arange(r // 2, dtype=np.float64)
        if kind == "dynamic":
            if r == 2:
                raise ValueError("dynamic scaling needs more than one pair")
            base = base * (s * s - (s - 1.0)) ** (r / (r - 2.0))
        freq = np.float64(base) ** (-2.0 * i / r)
        if kind == "linear":
            freq = freq / s
        elif kind == "yarn":
            m = int(scaling.pop("original_max_position_embeddings", max_position))
            kept, fast, slow = (float(scaling.pop(k, d)) for k, d in (("extrapolation_factor", 1.0), ("beta_fast", 32.0),
                                                                     ("beta_slow", 1.0)))
            if m < 1 or not fast > slow > 0:
                raise ValueError("yarn scaling needs beta_fast > beta_slow > 0 and a positive original length")
            pair = [r * math.log(m / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (fast, slow)]
            lo, hi = max(math.floor(pair[0]), 0), min(math.ceil(pair[1]), r - 1)
            ramp = np.clip((i - lo) / (hi - lo if hi > lo else 0.001), 0.0, 1.0)
            keep = (1.0 - ramp) * kept
            freq = freq / s * (1.0 - keep) + freq * keep
            self.attention_factor = float(scaling.pop("attn_factor", 1.0)) * (0.1 * math.log(s) + 1.0)
        if scaling:
            raise ValueError(f"entries of the scaling that {kind!r} has no use for: {sorted(scaling)}")
        self.frequencies = torch.from_numpy(freq)                         # radians per position, float64
        self._turns = freq / (2 * math.pi)
        self._pack()

    def _pack(self) -> None:
        # what the host's half of a call takes: address of the turns, pairs' values, layout, factor, head size
        self._packed = (self._turns.ctypes.data, self.rotary_dim, int(self.interleaved), self.attention_factor, self.head_dim)

    def __getstate__(self):
        return {k: v for k, v in self.__dict__.items() if k != "_packed"}

    def __setstate__(self, state) -> None:
        self.__dict__.update(state)
        self._pack()                                                      # (a copy's turns lie elsewhere)


def _stride(t: torch.Tensor, d: int) -> int:
    return t.stride(d) if t.shape[d] > 1 else 0      # (of a size of one it means nothing)


def _same_place(q: torch.Tensor, *others) -> None:
    device = q.device
    for t in others:
        if t is not None and t.device != device:
            raise ValueError("tensors must live on one GPU")


def _index(name: str, t: torch.Tensor, n: int, dtype) -> None:
    if t.dtype != dtype or t.dim() != 1 or t.shape[0] != n or (n > 1 and t.stride(0) != 1):
        raise ValueError(f"{name} must be a contiguous {str(dtype)[6:]} tensor [{n}]")


def _heads(name: str, t: torch.Tensor, like: Optional[torch.Tensor] = None) -> None:
    """[n, heads, dim] of a type there are kernels for, values of a head side by side."""
    if t.dim() != 3 or t.dtype not in _TYPES or (t.shape[2] > 1 and t.stride(2) != 1):
        raise ValueError(f"{name} must be a float16 or bfloat16 tensor [n, heads, dim] with contiguous heads")
    if like is not None and (t.dtype != like.dtype or t.shape[2] != like.shape[2] or t.shape[0] != like.shape[0]):
        raise ValueError(f"{name} must have the type, rows and head size of the others")


def _writable(name: str, t: torch.Tensor) -> None:
    """No two elements at one address: what a kernel writes side by side."""
    if t.is_contiguous():
        return
    upto = 1
    for stride, size in sorted((t.stride(d), t.shape[d]) for d in range(t.dim()) if t.shape[d] > 1):
        if stride < upto:
            raise ValueError(f"elements of {name} overlap")
        upto = stride * size


def _meet(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether an element of one may lie where one of the other does: exact where the larger strides step over what the
    smaller ones reach (slices of one projection, pools in one tensor), and else wherever the two's memory overlaps."""
    if not a.numel() or not b.numel():
        return False
    size, at = a.element_size(), b.data_ptr() - a.data_ptr()
    reach = [sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1 for t in (a, b)]
    if at >= reach[0] * size or -at >= reach[1] * b.element_size():
        return False
    if b.element_size() != size or at % size:
        return True
    steps: Dict[int, list] = {}                       # stride -> steps of a and of b
    for which, t in enumerate((a, b)):
        for n, s in zip(t.shape, t.stride()):
            if n > 1 and s:
                both = steps.setdefault(s, [0, 0])
                if both[which]:
                    return True
                both[which] = n - 1
    apart = {at // size}                              # from a row of a to one of b, by the strides so far; none: they do not meet
    for s in sorted(steps, reverse=True):
        na, nb = steps[s]
        reach = [reach[0] - na * s, reach[1] - nb * s]
        if s < max(reach):
            return True
        apart = {d - k * s for d in apart for k in (d // s, d // s + 1) if -nb <= k <= na}
        apart = {d for d in apart if -reach[1] < d < reach[0]}
        if not apart:
            return False
    return 0 in apart


def _apart(name: str, out: torch.Tensor, *others: Optional[torch.Tensor]) -> None:
    """What is written lies apart from what is read, and from what else is written."""
    for t in others:
        if t is not None and _meet(out, t):
            raise ValueError(f"{name} must be memory of its own")


def _itself(out: torch.Tensor, t: torch.Tensor) -> bool:
    return out.data_ptr() == t.data_ptr() and out.stride() == t.stride()


def _pages(name: str, t: torch.Tensor, q: torch.Tensor) -> None:
    if t.dim() != 4 or t.dtype != q.dtype or t.shape[3] != q.shape[2] or t.stride(3) != 1:
        raise ValueError(f"{name} must be [pages, kv_heads, page_size, dim] of q's type and head size, with contiguous heads")
    ps = t.shape[2]
    if ps < 8 or ps > 1024 or ps & (ps - 1):
        raise ValueError("a page must hold a power of two of tokens, from 8 to 1024")
    if not 1 <= t.shape[0] < 1 << 31 or not t.shape[1]:
        raise ValueError(f"{name} holds no pages")


def _status(dev: int) -> int:
    """Address of the device's status word for the paged cache; the current device's."""
    at = ops._page_status.get(dev)
    if at is None:
        at = _lib.lib().dz_page_status()
        if not at:
            raise RuntimeError("the library has no memory on the current device")
        ops._page_status[dev] = at
        _lib.host().arm(dev, at)
    return at


def _elsewhere(t: torch.Tensor) -> bool:
    """Whether the tensor's device is not the current one."""
    return t.get_device() != (ops._current_device() if ops._current_device is not None else torch.cuda.current_device())


@lru_cache(maxsize=1024)
def _attention_bytes(rows: int, heads: int, kv_heads: int, dim: int, page_size: int, pages_per_row: int) -> int:
    return _lib.lib().dz_paged_attention_bytes(rows, heads, kv_heads, dim, page_size, pages_per_row)


_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", torch.cuda.is_current_stream_capturing)


class _Space(NamedTuple):
    """What rows that are split over workgroups need: counters, all zero between calls, and room for the parts' sums."""
    counters: torch.Tensor
    work: torch.Tensor
    counters_at: int
    work_at: int
    work_bytes: int


_spaces: Dict[Tuple[int, int], _Space] = {}       # (device, stream)


# (device, stream) -> (capture, counters) of the graph that is being captured there
_captured: Dict[Tuple[int, int], Tuple[int, torch.Tensor]] = {}


def _parts_space(device: torch.device, need: int) -> _Space:
    """Calls on one stream follow each other and share theirs.  A graph may be replayed beside anything: it has counters of its
    own, cleared in it by the first captured call on a stream, and every captured call room of its own."""
    key = device.index, ops._stream()
    capture = _lib.lib().dz_capture_id(key[1]) if _capturing() else 0
    if capture:
        made = _captured.get(key)
        if made is None or made[0] != capture:
            made = _captured[key] = capture, torch.zeros(COUNTERS, dtype=torch.int32, device=device)
        counters, size = made[1], need
    else:
        space = _spaces.get(key)
        if space is not None and space.work_bytes >= need:
            return space
        counters = torch.zeros(COUNTERS, dtype=torch.int32, device=device) if space is None else space.counters
        size = max(need, 1 << 20)
    work = torch.empty(size, dtype=torch.uint8, device=device)
    space = _Space(counters, work, counters.data_ptr(), work.data_ptr(), size)
    if not capture:
        _spaces[key] = space
    return space


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_tables: torch.Tensor,
                    lengths: torch.Tensor, scale: Optional[float] = None, window: int = 0,
                    out: Optional[torch.Tensor] = None, shared: bool = False) -> torch.Tensor:
    """Attention of one new token per row (serving/csrc/attention):

        out[r, h] = softmax(scale q[r, h] . K)  V    over tokens max(0, n - window) .. n - 1 of row r, n = lengths[r]

    q [rows, heads, dim]; k_pages, v_pages [pages, kv_heads, page_size, dim], heads a multiple of kv_heads; token t of row r
    is token t % page_size of page block_tables[r, t // page_size].  block_tables int32 [rows, n], lengths int32 [rows], the
    new token counted.  scale defaults to dim ** -0.5; window 0: every token.  Any strides but the heads' values side by
    side and on multiples of 8 values (dim too, up to 256); pages of 8 to 1024 tokens, a power of two.

    A row of length 0 gives zeros.  Nothing behind a row's length is read, in the tables or in the pages, whatever
    is there; what it sees counts, and values there that are not finite give values that are not, in their row and head.  Several
    rows may share pages (`shared` says that most of what they see is: the same bits, up to 1.6 times as fast then, a
    tenth slower if it is not so; of one row nothing is), and several rows of one sequence at lengths of their own are a prompt's
    tokens.  A length beyond its table is cut; a page number outside the pool is read as page 0; either is reported through the
    status word.  The order of a row's sums follows the lengths of all rows of the call (the work is cut by them,
    256 rows at a time): the same lengths give the same bits."""
    if out is None:
        out = _lib.host().attend(q, k_pages, v_pages, block_tables, lengths, scale, window, shared)
        if out is not None:
            return out
    ops._need_cuda(q, k_pages, v_pages, block_tables, lengths, out)
    if _elsewhere(q):
        with torch.cuda.device(q.device):
            return paged_attention(q, k_pages, v_pages, block_tables, lengths, scale, window, out, shared)
    _same_place(q, k_pages, v_pages, block_tables, lengths, out)
    _heads("q", q)
    _pages("k_pages", k_pages, q)
    _pages("v_pages", v_pages, q)
    rows, heads, dim = q.shape
    pages, kv_heads, page_size, _ = k_pages.shape
    if v_pages.shape != k_pages.shape:
        raise ValueError("k_pages and v_pages must have one shape")
    if heads % kv_heads or not heads or heads > 4096 or dim % 8 or dim > MAX_DIM:
        raise ValueError(f"heads must be a multiple of kv_heads, up to 4096, and dim one of 8, up to {MAX_DIM}")
    if block_tables.dtype != torch.int32 or block_tables.dim() != 2 or block_tables.shape[0] != rows or (
            block_tables.shape[1] > 1 and block_tables.stride(1) != 1):
        raise ValueError(f"block_tables must be an int32 tensor [{rows}, n] with contiguous rows")
    _index("lengths", lengths, rows, torch.int32)
    width = block_tables.shape[1]
    if width * page_size > 1 << 30:
        raise ValueError("block_tables of more than 2^30 tokens a row")
    if window < 0:
        raise ValueError("window must be 0 (every token) or the number of tokens seen")
    if out is None:
        out = torch.empty((rows, heads, dim), dtype=q.dtype, device=q.device)
    else:
        _heads("out", out, q)
        if out.shape != q.shape:
            raise ValueError("out must have q's shape")
        _writable("out", out)
        _apart("out", out, q, k_pages, v_pages, block_tables, lengths)
    if rows == 0:
        return out
    need = _attention_bytes(rows, heads, kv_heads, dim, page_size, width)
    space = _parts_space(q.device, need) if need else None
    ks, vs = k_pages.stride(), v_pages.stride()
    args = _ATTENTION.pack(
        _ATTENTION.size, q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), block_tables.data_ptr(), lengths.data_ptr(),
        out.data_ptr(), space.work_at if need else 0, space.counters_at if need else 0, _status(q.get_device()), need, pages, _stride(q, 0), _stride(q, 1),
        ks[0] if pages > 1 else 0, ks[1] if kv_heads > 1 else 0, ks[2], vs[0] if pages > 1 else 0, vs[1] if kv_heads > 1 else 0,
        vs[2], _stride(out, 0), _stride(out, 1), block_tables.stride(0) if rows > 1 else 0, rows, heads, kv_heads, dim, page_size,
        width, min(int(window), (1 << 31) - 1), _TYPES[q.dtype], dim ** -0.5 if scale is None else scale, int(bool(shared)))
    _lib.check(_lib.lib().dz_paged_attention(args, ops._stream()), "dz_paged_attention")
    return out


def _rotate(q, k, v, positions, slots, rope, q_out, k_out, v_out, page_size, num_pages):
    tokens, heads, dim = q.shape
    paged = slots is not None
    strides = (lambda t: (_stride(t, 0), _stride(t, 1), t.stride(2))) if paged else (lambda t: (0, _stride(t, 1), _stride(t, 0)))
    args = _ROTARY.pack(
        _ROTARY.size, q.data_ptr(), 0 if k is None else k.data_ptr(), 0 if v is None else v.data_ptr(), q_out.data_ptr(),
        0 if k is None else k_out.data_ptr(), 0 if v is None else v_out.data_ptr(), positions.data_ptr(),
        slots.data_ptr() if paged else 0, 0 if rope is None else rope._packed[0], _status(q.get_device()) if paged else 0,
        num_pages, _stride(q, 0), _stride(q, 1), *((0, 0) if k is None else (_stride(k, 0), _stride(k, 1))),
        *((0, 0) if v is None else (_stride(v, 0), _stride(v, 1))), _stride(q_out, 0), _stride(q_out, 1),
        *((0, 0, 0) if k is None else strides(k_out)), *((0, 0, 0) if v is None else strides(v_out)),
        tokens, 0 if rope is None and q_out is q else heads, 0 if k is None else k.shape[1], dim, 0 if rope is None else rope.rotary_dim,
        0 if rope is None else int(rope.interleaved), page_size, _TYPES[q.dtype], 1.0 if rope is None else rope.attention_factor, 0)
    _lib.check(_lib.lib().dz_rotary(args, ops._stream()), "dz_rotary")


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, rope: RotaryPositions,
           out: Optional[Tuple[torch.Tensor, Optional[torch.Tensor]]] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """q [tokens, heads, dim] and k [tokens, kv_heads, dim] (or None) turned to `positions` (int64 [tokens], any
    value); returns new tensors, or writes `out` = (q, k): the inputs themselves (in place, as
    serving/csrc/pos_encoding does) or memory of their own.  Rows and heads may have any stride of an even number of values;
    with strides, sizes and half of rotary_dim multiples of eight, requests are four times as wide."""
    if out is None:
        made = _lib.host().rotate(q, k, None, positions, None, rope._packed, None, None, False)
        if made is not None:
            return made
    ops._need_cuda(q, k, positions)
    if _elsewhere(q):
        with torch.cuda.device(q.device):
            return rotary(q, k, positions, rope, out)
    _heads("q", q)
    if k is not None:
        _heads("k", k, q)
    _same_place(q, k, positions)
    if rope.head_dim != q.shape[2]:
        raise ValueError(f"heads of {q.shape[2]} values, positions made for {rope.head_dim}")
    _index("positions", positions, q.shape[0], torch.int64)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device), None if k is None else torch.empty(
            k.shape, dtype=k.dtype, device=k.device)
    else:
        if len(out) != 2 or out[0] is None or (out[1] is None) != (k is None):
            raise ValueError("out must be (q, k), with a tensor for each input")
        ops._need_cuda(*out)
        _same_place(q, *out)
        for n, (o, t) in enumerate(zip(out, (q, k))):
            if t is not None:
                _heads(f"out[{n}]", o, t)
                if o.shape != t.shape:
                    raise ValueError(f"out[{n}] must have its input's shape")
                _writable(f"out[{n}]", o)
                _apart(f"out[{n}]", o, None if _itself(o, t) else t, (k, q)[n], out[1 - n], positions)
        out = out[0], out[1]
    if q.shape[0] and (q.shape[1] or k is not None):
        _rotate(q, k, None, positions, None, rope, out[0], out[1], None, 8, 0)
    return out


def append_kv(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor,
              rope: Optional[RotaryPositions], k_pages: torch.Tensor, v_pages: torch.Tensor,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """A step's tokens stored in the cache, in one launch: k, turned, and v [tokens, kv_heads, dim] go to place
    slots[t] % page_size of page slots[t] // page_size of k_pages and v_pages [pages, kv_heads, page_size, dim]
    (serving/csrc/cache_kernels), and q [tokens, heads, dim], turned, is returned (or written to `out`, which
    may be q itself).  positions and slots int64 [tokens]; a negative slot stores nothing (a padded row: its q is turned all the
    same); one beyond the pages neither, and is reported through the status word.  rope None: nothing is turned, and q is
    returned as it is.  No two tokens may have one slot: what is there afterwards may be parts of either.  q, k and v lie
    outside the pages, and a q that is written lies apart from k and v.  Strides as for `rotary`."""
    if out is None or out is q:
        made = _lib.host().rotate(q, k, v, positions, slots, None if rope is None else rope._packed, k_pages, v_pages, out is q or rope is None)
        if made is not None:
            return made
    ops._need_cuda(q, k, v, positions, slots, k_pages, v_pages, out)
    if _elsewhere(q):
        with torch.cuda.device(q.device):
            return append_kv(q, k, v, positions, slots, rope, k_pages, v_pages, out)
    _same_place(q, k, v, positions, slots, k_pages, v_pages, out)
    _heads("q", q)
    _heads("k", k, q)
    _heads("v", v, q)
    if v.shape != k.shape:
        raise ValueError("k and v must have one shape")
    if rope is not None and rope.head_dim != q.shape[2]:
        raise ValueError(f"heads of {q.shape[2]} values, positions made for {rope.head_dim}")
    _pages("k_pages", k_pages, q)
    _pages("v_pages", v_pages, q)
    if k_pages.shape != v_pages.shape or k_pages.shape[1] != k.shape[1]:
        raise ValueError("k_pages and v_pages must have one shape, with k's heads")
    if _meet(k_pages, v_pages):
        raise ValueError("keys and values need pages of their own")
    _writable("k_pages", k_pages)
    _writable("v_pages", v_pages)
    turned = rope is not None or (out is not None and out is not q)          # whether q is read
    for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
        _apart(name, t, q if turned else None, k, v)
    _index("positions", positions, q.shape[0], torch.int64)
    _index("slots", slots, q.shape[0], torch.int64)
    if out is not None:
        _heads("out", out, q)
        if out.shape != q.shape:
            raise ValueError("out must have q's shape")
        _writable("out", out)
        if turned:
            _apart("out", out, None if _itself(out, q) else q, k, v, k_pages, v_pages, positions, slots)
    elif rope is None:
        out = q
    else:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if q.shape[0]:
        _rotate(q, k, v, positions, slots, rope, out, k_pages, v_pages, k_pages.shape[2], k_pages.shape[0])
    return out


def _pools_meet(at: Sequence[int], pages: int, stride: int, size: int) -> bool:
    """Whether pools that begin at these addresses share memory: they follow each other, or those that do not take turns within
    a page's stride."""
    at = sorted(at)
    run = at[:1]
    for a, b in zip(at, at[1:] + [at[-1] + pages * stride]):
        if b - a < (pages - 1) * stride + size:
            run.append(b)
            continue
        places = sorted((x - run[0]) % stride for x in run)
        if any(y - x < size for x, y in zip(places, places[1:] + [stride])):
            return True
        run = [b]
    return False


def copy_pages(pools: Union[torch.Tensor, Sequence[torch.Tensor]], pairs) -> None:
    """Page `a` copied over page `b` for every (a, b) of `pairs`, in every pool: in place, in one launch for up to 320 pairs
    and 128 pools (serving/csrc/cache_kernels).  pools: one tensor [pools, pages, ...], or a sequence of
    [pages, ...] of one shape, type and stride that share no memory, pages contiguous and of a multiple of 16 bytes.  pairs: host integers [n, 2],
    a tensor or a sequence; they are read before the call returns (a graph that captures the call copies the same
    pages at every replay).  All copies run side by side: no page may be written twice, or be both read and written."""
    if isinstance(pairs, list):
        pairs = np.asarray(pairs)
    if isinstance(pairs, np.ndarray) and pairs.dtype == np.int64:
        pairs = torch.from_numpy(pairs)
    stacked = isinstance(pools, torch.Tensor)
    if stacked and _lib.host().copy(pools, pairs):
        return
    if stacked:
        if pools.dim() < 2:
            raise ValueError("pools must be [pools, pages, ...]")
        first, n, step = (pools[0] if pools.shape[0] else None), pools.shape[0], pools.stride(0) * pools.element_size()
    else:
        pools = list(pools)
        first, n = (pools[0] if pools else None), len(pools)
        for t in pools:
            if t.shape != first.shape or t.dtype != first.dtype or t.stride() != first.stride() or t.device != first.device:
                raise ValueError("pools must have one shape, type, stride and device")
    if first is None:
        return
    ops._need_cuda(first)
    if _elsewhere(first):
        with torch.cuda.device(first.device):
            return copy_pages(pools, pairs)
    if first.dim() < 1:
        raise ValueError("a pool must be [pages, ...]")
    pages = first.shape[0]
    size = first.element_size() * math.prod(first.shape[1:])
    upto = 1
    for d in range(first.dim() - 1, 0, -1):
        if first.shape[d] > 1 and first.stride(d) != upto:
            raise ValueError("pages must be contiguous")
        upto *= first.shape[d]
    stride = first.stride(0) * first.element_size() if pages > 1 else size
    if size % 16 or stride % 16 or stride < size:
        raise ValueError("pages must be multiples of 16 bytes")
    if isinstance(pairs, torch.Tensor) and pairs.is_cuda:
        raise ValueError("pairs must be on the host")
    pairs = np.asarray(pairs)
    if pairs.size == 0:
        return
    if pairs.ndim != 2 or pairs.shape[1] != 2 or pairs.dtype.kind not in "iu":
        raise ValueError("pairs must be integers [n, 2]")
    if pairs.min() < 0 or pairs.max() >= pages:
        raise ValueError(f"pairs name pages outside [0, {pages})")
    pairs = np.ascontiguousarray(pairs, dtype=np.int32)
    written = set(pairs[:, 1].tolist())
    if len(written) < len(pairs) or not written.isdisjoint(pairs[:, 0].tolist()):
        raise ValueError("a page is written twice, or both read and written")
    at = [first.data_ptr() + i * step for i in range(n)] if stacked else [t.data_ptr() for t in pools]
    if _pools_meet(at, pages, stride, size):
        raise ValueError("pools share memory")
    _lib.check(_lib.lib().dz_copy_pages((C.c_void_p * n)(*at), n, stride, size, pages, pairs.ctypes.data, len(pairs), ops._stream()),
               "dz_copy_pages")
