"""Drop-in for the reference's ``kessie_attention`` module (KeSSie attention
backend for vLLM V1), with the fog actually applied.

The reference (kessie_attention.py:26-307) computes an additive fog bias
once per step (``_FogCache``) and passes it to vLLM's own attention as
``attn_bias``.  vLLM's FlashAttention implementation takes no such argument,
so the fog never reaches the scores; the reference also sizes the bias from
``key.shape[-2]``, the KV-head count of vLLM's [tokens, heads, dim] keys.
Here ``KeSSieAttentionImpl`` computes the attention itself with the paged
decode and ragged-chunk kernels of this library, the bias applied to the
scaled scores inside the kernels, per request of kv_len = its sequence
length:
    fb = int(kv_len * (1 - fog_start))
    bias(j) = -fog_alpha * (1 - j/fb)^2 for j < fb, 0 after,
    bias(j) = recall_boost at recalled positions
(the values of _FogCache._compute_into, kessie_attention.py:114-139).
Everything else (KV-cache write, metadata, cache layout) stays vLLM's:
the backend subclasses the FlashAttention backend and the impl delegates
to the wrapped FlashAttention impl.

Same names and state API as the reference: ``KeSSieAttentionState``,
``KESSIE_STATE``, ``_FogCache.get_fog_bias`` (the materialised
(1, 1, 1, kv_len) bias, built by a kernel), ``register_kessie_attention``,
``KeSSieAttentionBackend``, ``KeSSieAttentionImpl``.
"""

from __future__ import annotations

import logging
import os
import threading
from typing import NamedTuple, Optional, Sequence, Set, Tuple

import torch

from . import ops

logger = logging.getLogger("KeSSie.Attention")


class KeSSieAttentionState:
    """Thread-safe global fog parameters (kessie_attention.py:26-60)."""

    def __init__(self):
        self._lock = threading.Lock()
        self.fog_alpha: float = 0.5
        self.fog_start: float = 0.5
        self.prompt_len: int = 0
        self.recall_positions: Set[int] = set()
        self.recall_boost: float = 0.1
        self.enabled: bool = True
        self.generation: int = 0

    def update(self, fog_alpha=None, fog_start=None, prompt_len=None, recall_positions=None, recall_boost=None):
        with self._lock:
            if fog_alpha is not None:
                self.fog_alpha = fog_alpha
            if fog_start is not None:
                self.fog_start = fog_start
            if prompt_len is not None:
                self.prompt_len = prompt_len
            if recall_positions is not None:
                self.recall_positions = set(recall_positions)
            if recall_boost is not None:
                self.recall_boost = recall_boost
            self.generation += 1

    def get(self):
        with self._lock:
            return {"fog_alpha": self.fog_alpha, "fog_start": self.fog_start, "prompt_len": self.prompt_len,
                    "recall_positions": set(self.recall_positions), "recall_boost": self.recall_boost,
                    "enabled": self.enabled, "generation": self.generation}


KESSIE_STATE = KeSSieAttentionState()


class _FogCache:
    """The materialised bias of the reference API (kessie_attention.py:66-185):
    computed once per (generation, kv_len, device, dtype) into one of two
    ping-pong buffers by the library's bias kernel; later calls of the same
    generation return the same view.  The attention path below does not need
    it (the bias is evaluated inside the kernels)."""

    def __init__(self):
        self._gen = -1
        self._kv_len = 0
        self._buf = [None, None]
        self._active = 0
        self._alloc_len = 0
        self._device = None
        self._dtype = None
        self._view = None
        self._compute_lock = threading.Lock()

    def _ensure_alloc(self, kv_len, device, dtype):
        if self._alloc_len >= kv_len and self._device == device and self._dtype == dtype:
            return
        alloc = (max(kv_len, 2048) + 255) & ~255
        self._buf = [torch.zeros(alloc, device=device, dtype=dtype), torch.zeros(alloc, device=device, dtype=dtype)]
        self._alloc_len, self._device, self._dtype = alloc, device, dtype
        self._gen = -1
        self._view = None

    @staticmethod
    def _compute_into(buf, kv_len, fog_alpha, fog_start, recall_pos, recall_boost=0.1):
        """Bias of kv_len keys into buf[:kv_len] (kessie_attention.py:114-139)."""
        bias = ops.FogBias(fog_alpha, fog_start, recall_pos, recall_boost, dtype=buf.dtype, device=buf.device)
        ops.build_fog_bias(kv_len, bias, out=buf[:kv_len])

    def get_fog_bias(self, kv_len, device, dtype, state):
        """(1, 1, 1, kv_len) bias of the state's generation."""
        gen = state["generation"]
        if self._gen == gen and self._kv_len == kv_len and self._view is not None:
            return self._view
        with self._compute_lock:
            if self._gen == gen and self._kv_len == kv_len and self._view is not None:
                return self._view
            self._ensure_alloc(kv_len, device, dtype)
            self._active = 1 - self._active          # a new generation lands in the other buffer
            buf = self._buf[self._active]
            self._compute_into(buf, kv_len, state["fog_alpha"], state["fog_start"],
                               frozenset(state["recall_positions"]), state.get("recall_boost", 0.1))
            self._gen, self._kv_len = gen, kv_len
            self._view = buf[:kv_len].view(1, 1, 1, kv_len)
            return self._view


def _fog_active(state) -> bool:
    """The reference's switch (kessie_attention.py:276-277)."""
    return bool(state["enabled"]) and state["fog_alpha"] > 0 and state["prompt_len"] > 0


class _BiasCache:
    """FogBias (device recall bitmap included) of the current generation."""

    def __init__(self):
        self._lock = threading.Lock()
        self._key = None
        self._bias = None

    def get(self, state, dtype, device) -> "ops.FogBias":
        key = (state["generation"], dtype, device)
        with self._lock:
            if self._key != key:
                self._bias = ops.FogBias(state["fog_alpha"], state["fog_start"], state["recall_positions"],
                                         state.get("recall_boost", 0.1), dtype=dtype, device=device)
                self._key = key
            return self._bias


_BIAS_CACHE = _BiasCache()
_FOG_CACHE = _FogCache()


class QueryRun(NamedTuple):
    """Neighbouring requests [first, end) of a step, from row `row` of its
    tokens on, that all have one new token (decodes) or none of which has."""
    first: int
    end: int
    row: int
    decodes: bool


def query_runs(starts: Sequence[int], most: Optional[int] = None) -> Tuple[QueryRun, ...]:
    """The runs of a step, from the offsets of its requests' tokens (on the
    host); none of them where there are more than `most`."""
    starts = torch.as_tensor(starts, device="cpu")
    one = starts.diff() == 1
    if one.numel() == 0:
        return ()
    firsts = [0] + ((one[1:] != one[:-1]).nonzero().flatten() + 1).tolist()
    if most is not None and len(firsts) > most:
        return ()
    return tuple(QueryRun(f, e, int(starts[f]), bool(one[f])) for f, e in zip(firsts, firsts[1:] + [one.numel()]))


# A mixed step's decodes go to the paged decode, apart from its chunks, when there is one run of each and the decodes
# have at least this many (request, KV head) pairs an SM: the ragged call pays for the start and end of each of those
# tiles, which few of them hide in the chunks' time and many do not.  GPU time a layer, one call against two (bf16,
# 32 / 8 heads of 128): 64 decodes over 2,000 keys + a prompt of 512 150 against 126 us, 256 over 500 + 512 209 / 162,
# 64 over 32,000 + 2,048 1,576 / 1,336; 32 over 500 + 512 58 / 72, 16 over 8,000 + 16 105 / 112.
_SPLIT_TILES = 3


class KeSSieAttentionImpl:
    """Per-layer attention: with the fog active, a decode step runs in the paged
    decode and any other step (prompt chunks, drafts, decodes mixed) in one
    ragged-chunk call, or with many decodes in one call of each, none reading a
    length back to the host, with the fog bias applied to the scores;
    otherwise (fog off, profiling run, features the kernels do not cover) the
    wrapped vLLM implementation runs.  Attributes and methods not defined here
    (e.g. the KV-cache write) are the wrapped implementation's."""

    def __init__(self, *args, _inner_impl=None, **kwargs):
        if _inner_impl is None:
            if not HAS_VLLM:
                raise RuntimeError("KeSSieAttentionImpl needs vLLM or an injected implementation")
            _inner_impl = KeSSieAttentionBackend._get_original().get_impl_cls()(*args, **kwargs)
        object.__setattr__(self, "_inner", _inner_impl)
        inner = _inner_impl
        self._num_heads = int(inner.num_heads)
        self._num_kv_heads = int(getattr(inner, "num_kv_heads", inner.num_heads))
        self._head_size = int(inner.head_size)
        self._scale = float(inner.scale)
        sw = getattr(inner, "sliding_window", None)
        if sw is None or (isinstance(sw, (tuple, list)) and sw[0] < 0):
            self._window = 0
        elif isinstance(sw, (tuple, list)):
            self._window = int(sw[0]) + 1                 # vLLM keeps (window - 1, 0)
        else:
            self._window = int(sw)

    def __getattr__(self, name):
        return getattr(object.__getattribute__(self, "_inner"), name)

    # ------------------------------------------------------------------ dispatch
    def _kernels_cover(self, query, kv_cache, output, output_scale) -> bool:
        inner = self._inner
        if output is None or output_scale is not None or kv_cache is None or not query.is_cuda:
            return False
        if query.dtype not in (torch.bfloat16, torch.float16) or kv_cache.dtype != query.dtype:
            return False
        if self._head_size not in (64, 128) or self._num_heads % self._num_kv_heads:
            return False
        if self._num_heads // self._num_kv_heads > 16:
            return False
        if getattr(inner, "alibi_slopes", None) is not None or getattr(inner, "sinks", None) is not None:
            return False
        if getattr(inner, "logits_soft_cap", 0) not in (None, 0, 0.0):
            return False
        return kv_cache.dim() == 5 and kv_cache.shape[0] == 2

    def forward(self, layer, query, key, value, kv_cache, attn_metadata, output=None, output_scale=None,
                output_block_scale=None):
        state = KESSIE_STATE.get()
        if attn_metadata is None or not _fog_active(state) or \
                not self._kernels_cover(query, kv_cache, output, output_scale):
            return self._inner.forward(layer, query, key, value, kv_cache, attn_metadata, output, output_scale,
                                       output_block_scale)
        return self._fog_forward(query, kv_cache, attn_metadata, output, state)

    @staticmethod
    def _check_lengths(md, capacity):
        """Raise for a request of several new tokens that is longer than its
        row of the block table.  Called where vLLM's bound on the lengths is
        above the row's, so that the lengths themselves are read by the host
        only then (in a capture they cannot be: the kernel cuts them and
        records it in the device status)."""
        if torch.cuda.is_current_stream_capturing():
            return
        starts, lens = md.query_start_loc.tolist(), md.seq_lens.tolist()
        for first, end, n in zip(starts, starts[1:], lens):
            if end - first > 1 and n > capacity:
                raise ValueError(f"max_kv_len {n} exceeds the block table capacity {capacity}")

    def _fog_forward(self, query, kv_cache, md, output, state):
        n = int(md.num_actual_tokens)
        Hq, D = self._num_heads, self._head_size
        q = query[:n].view(n, Hq, D)
        out = output[:n].view(n, Hq, D)
        key_cache, value_cache = kv_cache.unbind(0)      # [num_blocks, block_size, Hkv, D] each
        bias = _BIAS_CACHE.get(state, query.dtype, query.device)
        bt, sl = md.block_table, md.seq_lens
        kw = dict(window_size=self._window, sm_scale=self._scale, fog_alpha=0.0, bias=bias)
        if int(md.max_query_len) == 1:                 # decode step: one launch for the batch
            ops.paged_fog_decode(q, key_cache, value_cache, bt[:n], sl[:n], out=out, **kw)
            return output
        # a mixed step (prompt chunks, drafts, decodes): one call for the batch, or two; lengths read on the device
        B = sl.shape[0]
        capacity = bt.shape[1] * key_cache.shape[1]
        if (getattr(md, "max_seq_len", None) or 0) > capacity:
            self._check_lengths(md, capacity)
        for run in self._launches(md, B, capacity, key_cache.shape[1], out):
            if run.decodes:
                rows, reqs = slice(run.row, run.row + run.end - run.first), slice(run.first, run.end)
                ops.paged_fog_decode(q[rows], key_cache, value_cache, bt[reqs], sl[reqs], out=out[rows], **kw)
                continue
            for b in range(run.first, run.end, ops.MAX_CHUNK_SEQUENCES):     # one call, but for the largest batches
                e = min(b + ops.MAX_CHUNK_SEQUENCES, run.end)
                ops.paged_fog_chunks(q, key_cache, value_cache, bt[b:e], md.query_start_loc[b:e + 1], sl[b:e], out=out,
                                     **kw)
        return output

    def _launches(self, md, B, capacity, page_size, out):
        """The calls of a mixed step of B requests: all of them in one
        ragged-chunk call, or the decodes apart in the paged decode.  The
        latter takes the metadata builder's host copy of the offsets; a capture
        holds for other offsets too, and is one call."""
        runs = getattr(md, "query_runs", None)
        whole = (QueryRun(0, B, 0, False),)
        if not runs or len(runs) != 2 or runs[-1].end != B or torch.cuda.is_current_stream_capturing():
            return whole
        tiles = sum(r.end - r.first for r in runs if r.decodes) * self._num_kv_heads
        sms = torch.cuda.get_device_properties(md.seq_lens.device).multi_processor_count
        if tiles < _SPLIT_TILES * sms:
            return whole
        if page_size > 256 or tiles * (capacity // 16) > 1 << 30 or not out.is_contiguous():      # the decode's limits
            return whole
        return runs


# ----------------------------------------------------------------- vLLM registration
try:
    from vllm.v1.attention.backends.flash_attn import FlashAttentionBackend as _FlashAttentionBackend
    HAS_VLLM = True
except Exception:                                      # pragma: no cover - depends on the vLLM build
    _FlashAttentionBackend = None
    HAS_VLLM = False

if HAS_VLLM:
    class KeSSieAttentionBackend(_FlashAttentionBackend):
        """FlashAttention backend whose implementation applies the fog
        (kessie_attention.py:228-260); metadata and cache layout are
        FlashAttention's, and so is the builder but for a mixed step's runs."""

        @classmethod
        def _get_original(cls):
            return _FlashAttentionBackend

        @staticmethod
        def get_name() -> str:
            return "KeSSie"

        @staticmethod
        def get_impl_cls():
            return KeSSieAttentionImpl

        @staticmethod
        def get_builder_cls():
            return KeSSieMetadataBuilder

    class KeSSieMetadataBuilder(_FlashAttentionBackend.get_builder_cls()):
        """FlashAttention's builder; the metadata of a mixed step carries its
        runs of decodes and chunks, from vLLM's host copy of the offsets."""

        def build(self, common_prefix_len, common_attn_metadata, fast_build=False):
            md = super().build(common_prefix_len, common_attn_metadata, fast_build)
            starts = getattr(common_attn_metadata, "query_start_loc_cpu", None)
            if starts is not None and common_attn_metadata.max_query_len > 1:
                md.query_runs = query_runs(starts, 2)           # of more the attention makes no use
            return md
else:
    class KeSSieAttentionBackend:                      # pragma: no cover
        pass


def register_kessie_attention() -> bool:
    """Register the KeSSie backend in place of FLASH_ATTN; call before the
    engine is created (kessie_attention.py:188-212)."""
    if not HAS_VLLM:
        logger.warning("vLLM V1 attention registry not available")
        return False
    try:
        from vllm.v1.attention.backends.registry import AttentionBackendEnum, register_backend
    except ImportError:
        logger.warning("vLLM V1 attention registry not available")
        return False
    target = AttentionBackendEnum.FLASH_ATTN
    os.environ["_KESSIE_ORIGINAL_ATTN_PATH"] = target.value
    register_backend(target, "kessie_b200.kessie_attention.KeSSieAttentionBackend")
    logger.info("KeSSie attention registered (wrapping %s)", target.value)
    return True
