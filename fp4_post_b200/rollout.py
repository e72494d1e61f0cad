"""What generating takes besides the projections: rotary positions, a key-value cache in pages with attention over it, and sampling.

    Rotary       rotary positions of queries and keys: both layouts, a part of the head, scaled for long contexts; differentiable
    PagedCache   keys and values of many sequences in pages that they may share: reserve, append (with the rotary positions), attend (one new
                 token for each sequence), fork, free, compact
    sample       one token for each row of logits, by given random numbers

A decode step of a layer is

    q = cache.append(layer, q, k, v, rotary=rotary)        # rotate, write k and v behind each sequence
    o = cache.attend(layer, q)

between one cache.reserve(slots, 1) for all layers and one sample() of the logits; Decoder.generate (decoder.py) is that loop.  All state is on
the device (page tables, lengths, reference counts), so that a step needs no word from the host and can be captured in a CUDA graph.

Kernels of this library (csrc/rotary.cu, paged_cache.cu, paged_attention.cu, sample.cu) behind native calls (csrc/rollout_host.cpp); CUDA
tensors only, nothing here computes on the CPU.  A call runs on the current stream of its tensors' device.  They are no operations of
torch: forward-mode derivatives, traces and tensor subclasses that dispatch by themselves are refused, and, but for Rotary, so are tensors that
require a gradient while it is recorded.

The reference leaves all of this to the Hugging Face model that it generates with (src/grpo/grpo.py:673-693).
"""
from __future__ import annotations

import math
import operator
from typing import Optional, Union

import torch

from . import cabi

SCALINGS = ("linear", "llama3", "yarn")


def rotary_frequencies(rotary_dim: int, theta: float = 1e4, scaling: Optional[dict] = None):
    """(angles per position of the rotary_dim / 2 pairs, as Python floats; what rotated values are multiplied by).

    Pair i turns by theta^(-2i / rotary_dim) per position.  scaling, by its "type":
      linear   all frequencies / factor
      llama3   pairs of wavelengths below original_max_position / high_freq_factor stay, those above original_max_position / low_freq_factor are
               divided by factor, those between are interpolated in 1 / wavelength
      yarn     pairs that turn more than beta_fast (32) times over original_max_position stay, those that turn less than beta_slow (1) times are
               divided by factor, those between are interpolated by their index; magnitude 0.1 ln(factor) + 1, or attention_factor"""
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be a positive even number, not {rotary_dim}")
    if not (theta > 1.0 and math.isfinite(theta)):
        raise ValueError(f"theta must be finite and above 1, not {theta}")
    plain = [theta ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)]
    if scaling is None:
        return plain, 1.0
    known = dict(scaling)
    kind, factor = known.pop("type", None), float(known.pop("factor", 0.0))
    if kind not in SCALINGS:
        raise ValueError(f"scaling['type'] must be one of {', '.join(SCALINGS)}, not {kind!r}")
    if not (factor > 0.0 and math.isfinite(factor)):
        raise ValueError(f"scaling['factor'] must be positive, not {factor}")

    def number(name, default=None):
        value = known.pop(name, default)
        if value is None or not (float(value) > 0.0 and math.isfinite(value)):
            raise ValueError(f"scaling['{name}'] must be a positive number for {kind}, not {value!r}")
        return float(value)

    magnitude = 1.0
    if kind == "linear":
        scaled = [f / factor for f in plain]
    elif kind == "llama3":
        low, high, original = number("low_freq_factor", 1.0), number("high_freq_factor", 4.0), number("original_max_position")
        if low >= high:
            raise ValueError(f"scaling: low_freq_factor {low} must be below high_freq_factor {high}")
        scaled = []
        for f in plain:
            mix = min(1.0, max(0.0, (original * f / (2.0 * math.pi) - low) / (high - low)))
            scaled.append((1.0 - mix) * f / factor + mix * f)
    else:
        fast, slow, original = number("beta_fast", 32.0), number("beta_slow", 1.0), number("original_max_position")
        magnitude = number("attention_factor", 0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0)

        def index_of(turns):         # of the pair that turns so often over the original length
            return rotary_dim * math.log(original / (turns * 2.0 * math.pi)) / (2.0 * math.log(theta))
        first, last = max(math.floor(index_of(fast)), 0), min(math.ceil(index_of(slow)), rotary_dim - 1)
        scaled = []
        for i, f in enumerate(plain):
            mix = min(1.0, max(0.0, (i - first) / max(last - first, 1e-3)))
            scaled.append(f / factor * mix + f * (1.0 - mix))
    if known:
        raise ValueError(f"scaling: {kind} does not know {', '.join(sorted(known))}")
    return scaled, magnitude


class Rotary:
    """Rotary positions of the first rotary_dim (None: all) of head_dim elements.

    interleaved: pairs are neighbours (2i, 2i + 1); else they lie half of rotary_dim apart (i, rotary_dim / 2 + i).  theta, scaling: see
    rotary_frequencies.  Angles are formed from the positions in whole numbers, exactly modulo a turn: there is no table and no longest position.
    Frequencies are 64-bit floats, off by up to 2^-53 turns per position, which is below the rounding of fp32 up to position 2^26.

        q, k = rotary(q, k, positions)

    q [..., heads, head_dim] and k [..., kv_heads, head_dim] (or None), both bfloat16 or both float32, of any strides over a dense last dimension;
    positions int32 or int64, of the leading dimensions' shape or one that broadcasts to it (None: 0, 1, ... along the last of them).  Computed in
    fp32, rounded once.  Results are contiguous.  Differentiable, any number of times, in q and k; both directions can be captured in a CUDA graph (a
    backward pass while no eager graph of the same leaves is kept: see graphs.py)."""

    def __init__(self, head_dim: int, *, theta: float = 1e4, rotary_dim: Optional[int] = None, interleaved: bool = False,
                 scaling: Optional[dict] = None, device: Union[str, torch.device] = "cuda"):
        self.head_dim = int(head_dim)
        self.rotary_dim = self.head_dim if rotary_dim is None else int(rotary_dim)
        if self.head_dim <= 0 or self.head_dim % 8 or self.head_dim > 256:
            raise ValueError(f"head_dim must be a multiple of 8 up to 256, not {head_dim}")
        if self.rotary_dim > self.head_dim:
            raise ValueError(f"rotary_dim {rotary_dim} is more than head_dim {head_dim}")
        self.interleaved = bool(interleaved)
        frequencies, self.magnitude = rotary_frequencies(self.rotary_dim, theta, scaling)
        # fractions of a turn in 64 bits: a product with a position, taken modulo 2^64, is the angle modulo a turn
        bits = [round(f / (2.0 * math.pi) * 2.0 ** 64) % 2 ** 64 for f in frequencies]
        with torch.inference_mode(False):        # (one made while generating is there to train with afterwards: an inference tensor cannot be saved for a backward pass)
            self.turns = torch.tensor([b - 2 ** 64 if b >= 2 ** 63 else b for b in bits], dtype=torch.int64, device=device)

    def __call__(self, q: torch.Tensor, k: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None):
        """(q, k) turned; q alone where there is no k."""
        if isinstance(q, torch.Tensor) and q.dim() and q.shape[-1] != self.head_dim:
            raise ValueError(f"q has heads of {q.shape[-1]} elements, not {self.head_dim}")
        q, k = cabi.rollout_host().rotary(q, k, positions, self.turns, self.magnitude, self.rotary_dim, self.interleaved)
        return q if k is None else (q, k)


class PagedCache:
    """Keys and values of up to `sequences` sequences of up to max_length tokens, in `pages` pages of page_size tokens for all layers.

        pool     [pages, layers, 2, kv_heads, page_size, head_dim]: bfloat16, or float8_e4m3fn with scales
        tables   [sequences, width] int32: each sequence's pages in order, -1 behind them
        lengths  [sequences] int32
        refs     [pages] int32: how many tables hold a page; 0 is a free one
        scales   [layers, 2, kv_heads] float32 (8-bit pools): an element stands for itself times its scale
        status   [1] int32: see below

    A sequence is named by its row ("slot").  Free pages are taken lowest first.  head_dim is a multiple of 8 up to 256,
    page_size of 16.  Everything is on the device and every call asynchronous: a call that cannot be done (too few
    free pages, a slot out of range or given twice, a sequence that would be too long, a fork onto one that is not empty) does nothing at all and leaves its reason in
    `status`, the first one; check() reads it.  Slots are int32 or int64 tensors on the device (lists are copied there); a negative one stands for nobody, so
    that padded batches can be given as they are.  Calls on one cache belong on one stream, or behind one another by events."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, *, pages: int, sequences: int, max_length: int, page_size: int = 16,
                 dtype: torch.dtype = torch.bfloat16, scales: Optional[torch.Tensor] = None, device: Union[str, torch.device] = "cuda"):
        device = torch.device(device)
        if page_size <= 0:
            raise ValueError(f"page_size must be a multiple of 16, not {page_size}")
        pool = torch.zeros((pages, layers, 2, kv_heads, page_size, head_dim), dtype=dtype, device=device)
        if dtype == torch.float8_e4m3fn and scales is None:
            scales = torch.ones((layers, 2, kv_heads), dtype=torch.float32, device=device)
        self._set(pool, torch.full((sequences, -(-max_length // page_size)), -1, dtype=torch.int32, device=device),
                  torch.zeros(sequences, dtype=torch.int32, device=device), torch.zeros(pages, dtype=torch.int32, device=device), scales)

    @classmethod
    def of(cls, pool: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor, refs: torch.Tensor, *, scales: Optional[torch.Tensor] = None) -> "PagedCache":
        """A cache of tensors that are there already; they are used as they are, and have to agree with one another.  Their memory is looked up at each
        call (a pool's storage may be given back for a while), what they are is not to change; a captured graph keeps the addresses that it was captured with.  The status, and which
        sequences reserve() could not lengthen, are this cache's own: two caches of the same tensors do not know one another's."""
        self = cls.__new__(cls)
        self._set(pool, tables, lengths, refs, scales)
        return self

    def _set(self, pool, tables, lengths, refs, scales):
        if not isinstance(pool, torch.Tensor):
            raise TypeError(f"pool must be a tensor, not {type(pool).__name__}")
        with torch.inference_mode(False):        # (check() writes to it in whatever mode)
            status = torch.zeros(1, dtype=torch.int32, device=pool.device)
        # by sequence, whether the last reserve() that named it could not be done
        refused = torch.zeros(lengths.numel() if isinstance(lengths, torch.Tensor) else 0, dtype=torch.int32, device=pool.device)
        self._handle = cabi.rollout_host().cache(pool, tables, lengths, refs, scales, status, refused)
        self._tensors = (pool, tables, lengths, refs, scales, status)
        self._host = cabi.rollout_host()

    pool = property(lambda self: self._tensors[0])
    tables = property(lambda self: self._tensors[1])
    lengths = property(lambda self: self._tensors[2])
    refs = property(lambda self: self._tensors[3])
    scales = property(lambda self: self._tensors[4])
    status = property(lambda self: self._tensors[5])
    layers = property(lambda self: self.pool.shape[1])
    kv_heads = property(lambda self: self.pool.shape[3])
    page_size = property(lambda self: self.pool.shape[4])
    head_dim = property(lambda self: self.pool.shape[5])
    sequences = property(lambda self: self.tables.shape[0])
    max_length = property(lambda self: self.tables.shape[1] * self.page_size)

    def _index(self, t):
        """Slots, counts or positions; what is not a tensor is copied to the device, and has to be whole numbers (torch cuts others)."""
        return t if t is None or isinstance(t, torch.Tensor) else torch.tensor([operator.index(i) for i in t], dtype=torch.int64, device=self.pool.device)

    def reserve(self, slots=None, counts: Union[int, torch.Tensor, list] = 1) -> None:
        """Lengthens the sequences `slots` (None: all) by `counts` tokens, one number or one for each, with pages for them.  Where that cannot be done, append()
        without positions writes nothing to any of them until a reserve() for it goes through."""
        one = counts if isinstance(counts, int) else None
        if one is None and not isinstance(counts, torch.Tensor):
            try:
                one = operator.index(counts)
            except TypeError:                # (one for each)
                pass
        self._host.reserve(self._handle, self._index(slots), None if one is not None else self._index(counts), one or 0)

    def append(self, layer: int, q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, slots=None, positions=None, *,
               rotary: Optional[Rotary] = None) -> Optional[torch.Tensor]:
        """Writes keys and values of reserved tokens, the keys (and q) turned by their rotary positions first; returns the queries.

        q [tokens, heads, head_dim] (or None), k and v [tokens, kv_heads, head_dim], bfloat16.  Token i belongs to sequence slots[i] (None: i) at
        positions[i] (None: its last one, and the token is not written where the reserve() that was to make room for it could not be done; its query is turned as
        at the last position then).  A token of no sequence is not written, and its query comes back as zeros; one at a position that is not
        reserved is not written.  8-bit pools take round to nearest of x / scale, saturating.  A page that several sequences hold changes for all of
        them.  Two tokens of one call must not go to the same place: one of them is there afterwards."""
        if rotary is None:
            return self._host.append(self._handle, layer, q, k, v, self._index(slots), self._index(positions), None, 1.0, 0, False)
        if rotary.head_dim != self.pool.shape[5]:
            raise ValueError(f"rotary positions of heads of {rotary.head_dim} elements, and a cache of {self.pool.shape[5]}")
        return self._host.append(self._handle, layer, q, k, v, self._index(slots), self._index(positions), rotary.turns, rotary.magnitude, rotary.rotary_dim, rotary.interleaved)

    def attend(self, layer: int, q: torch.Tensor, slots=None, *, scale: Optional[float] = None, return_lse: bool = False):
        """softmax(scale q K^T) V of one token for each row over all keys of its sequence: bfloat16, shaped like q [rows, heads, head_dim].

        Row i belongs to sequence slots[i] (None: i).  heads is a multiple of kv_heads, at most 1024 times; query head h reads key-value head h // (heads / kv_heads).  scale:
        1 / sqrt(head_dim) where None.  A row without keys, or of no sequence, is zeros.  Products on the tensor core, statistics and sums in fp32; the
        result does not depend on the other rows of the call beyond where its keys are split.  return_lse: also the logarithm of each row's sum of
        exp(scale q k), float32 [rows, heads] (-inf without keys)."""
        out, lse = self._host.attend(self._handle, layer, q, self._index(slots), self.pool.shape[5] ** -0.5 if scale is None else scale, return_lse)
        return (out, lse) if return_lse else out

    def fork(self, src, dst, *, share: bool = True) -> None:
        """Makes the empty sequences `dst` what `src` are: whole pages are held by both and what the last page is filled with is copied; with share=False
        all is copied.  One source may be given many times (a prompt and its group of answers)."""
        self._host.fork(self._handle, self._index(src), self._index(dst), share)

    def free(self, slots=None) -> None:
        """Empties the sequences `slots` (None: all).  Pages that nobody else holds are free."""
        self._host.release(self._handle, self._index(slots))

    def compact(self) -> torch.Tensor:
        """Moves the pages that are held to the front of the pool, and returns how many they are (int32 [1], on the device): pool[:n] is all
        there is to keep, save or send."""
        return self._host.compact(self._handle)

    def free_pages(self) -> int:
        """How many pages are free (reads the device)."""
        return int((self.refs == 0).sum())

    def check(self) -> None:
        """Raises if a call since the last check could not be done (reads the device)."""
        code = int(self.status)
        if code:
            self.status.zero_()
            raise RuntimeError(f"paged cache: {cabi.STATUS_TEXT.get(code, code)}")


Numbers = Union[float, torch.Tensor]


def sample(logits: torch.Tensor, u: torch.Tensor, *, temperature: Numbers = 1.0, top_k: Union[int, torch.Tensor] = 0, top_p: Numbers = 1.0,
           min_p: Numbers = 0.0, logprobs: bool = False):
    """One token (int64) for each row of logits [rows, vocab], bfloat16 or float32, by u [rows] in [0, 1), float32 or float64.

    With w = exp((x - max x) / temperature) and the tokens in order of their logits, equal ones by index: the first top_k (0: all) are kept; of them
    the shortest front that has top_p of their weights; of them those with w >= min_p; always the first.  The token is the first one, by index, up to
    which the kept weights exceed u times their sum.  temperature 0 takes the first of the order.  Weights are fp32, their sums exact or 64 bits wide: the
    same inputs give the same tokens, in whatever batch.

    Each parameter is a number or a tensor with one for each row (float32, top_k int32).  -inf and NaN are never taken.  A row with nothing else, or with a
    parameter in a tensor (or a u) out of its range, gives -1.  logprobs=True: also log softmax(logits / temperature) of the tokens over the
    whole vocabulary, float32 [rows] (temperature 0: of the logits as they are; NaN beside -1): what dense.token_logprobs gives for them."""
    token, logprob = cabi.rollout_host().sample(logits, u, temperature, top_k, top_p, min_p, logprobs)
    return (token, logprob) if logprobs else token
