"""Rotary position embedding, host side (reference: llama/positional_embeddings.py:5-36, 94-122).

`inv_freq` is a registered buffer exactly as in the reference (it appears in the state dict as
`...self_attn.rotary_emb.inv_freq`).  The cos/sin cache is kept as fp32 half tables [S, d/2] -- the
reference rounds its tables to bf16 when precision is bf16 (:33-35); keeping fp32 is closer to the
exact rotation and is what the parity tests compare against.

Not in the reference: `rotary_dim` (the part of a head that is turned), `interleaved` (pairs of neighbours instead of halves) and `scaling` (frequencies for
contexts longer than those of pre-training).  Such positions have no tables: their angles are computed where they are used, in 64 bits, and position ids may
lie anywhere.
"""
import math

import torch

from . import functional as F_
from . import kernels as K


_SCALINGS = {"linear": ("factor",), "dynamic": ("factor", "original_length"), "yarn": ("factor", "original_length")}
_SCALING_OPTIONS = {"linear": (), "dynamic": ("length",), "yarn": ("beta_fast", "beta_slow", "attention_factor")}


def scaled_frequencies(inv_freq, base, scaling, length):
    """(frequencies in fp64, what sines and cosines are multiplied by) of `inv_freq` [n] = base^(-j / n) under a scaling, a dict with a "type":

    linear   all divided by "factor"
    dynamic  a larger base for texts of `length` (or its own "length") tokens, where that is above "original_length": base ((factor length / original_length) - (factor - 1))^(n / (n - 1))
    yarn     divided by "factor" where a wave turns less than "beta_slow" (1) times in "original_length", as they are where it turns more than "beta_fast" (32) times, in between by a
             line over the index (Peng, Quesnelle, Fan, Shippole, "YaRN: efficient context window extension of large language models", 2023); "attention_factor"
             (0.1 ln factor + 1)"""
    n, device = inv_freq.numel(), inv_freq.device
    stretch, factor = _stretch(n, base, scaling, device)
    if _goes_by_length(scaling):
        stretch = _dynamic_stretch(stretch, scaling, length)
    return inv_freq.double() * stretch, factor


def _goes_by_length(scaling):
    return scaling is not None and scaling["type"] == "dynamic" and not scaling.get("length")


def _dynamic_stretch(exponents, scaling, length):
    factor, original = float(scaling["factor"]), float(scaling["original_length"])
    return 1.0 if length <= original else (factor * length / original - (factor - 1)) ** exponents


def _stretch(n, base, scaling, device):
    """(what n frequencies are multiplied by, in fp64, or a dynamic scaling's exponents where the length is not known yet; what sines and cosines are multiplied by)"""
    j = torch.arange(n, dtype=torch.float64, device=device)
    if scaling is None:
        return torch.ones_like(j), 1.0
    kind, factor = scaling["type"], float(scaling["factor"])
    if kind == "linear":
        return torch.full_like(j, 1 / factor), 1.0
    if kind == "dynamic":
        exponents = j / -max(n - 1, 1)  # (one frequency stays as it is)
        return exponents if _goes_by_length(scaling) else torch.ones_like(j) * _dynamic_stretch(exponents, scaling, scaling["length"]), 1.0
    original = float(scaling["original_length"])

    def index_of(turns):  # of the wave that turns so often in the original length
        return n * math.log(original / (turns * 2 * math.pi)) / math.log(base)

    low, high = max(math.floor(index_of(scaling.get("beta_fast", 32))), 0), min(math.ceil(index_of(scaling.get("beta_slow", 1))), 2 * n - 1)
    slow = ((j - low) / max(high - low, 1e-3)).clamp(0, 1)
    attention_factor = scaling.get("attention_factor")
    return slow / factor + (1 - slow), 0.1 * math.log(factor) + 1 if attention_factor is None else float(attention_factor)


def _checked_scaling(scaling):
    if scaling is None:
        return None
    kind = scaling.get("type")
    if kind not in _SCALINGS:
        raise NotImplementedError("scaling type %r: %s are built" % (kind, ", ".join(_SCALINGS)))
    unknown = set(scaling) - {"type", *_SCALINGS[kind], *_SCALING_OPTIONS[kind]}
    missing = set(_SCALINGS[kind]) - set(scaling)
    if unknown or missing:
        raise ValueError("scaling %r: %s" % (kind, "; ".join(["unknown %s" % n for n in sorted(unknown)] + ["%s is missing" % n for n in sorted(missing)])))
    if not float(scaling["factor"]) >= 1 or ("original_length" in scaling and not scaling["original_length"] > 0):
        raise ValueError("scaling: a factor of 1 or more, an original_length above 0")
    return dict(scaling)


def _capturing(device):
    return device.type == "cuda" and torch.cuda.is_current_stream_capturing()


class RotaryEmbedding(torch.nn.Module):
    def __init__(self, dim, base=10000, precision=torch.half, scale_factor=1.0, rotary_dim=None, interleaved=False, scaling=None):
        super().__init__()
        rotary_dim = dim if rotary_dim is None else rotary_dim
        if not 0 < rotary_dim <= dim or rotary_dim % 2:
            raise ValueError("rotary_dim must be even and at most the head's width, got %r of %r" % (rotary_dim, dim))
        inv_freq = 1.0 / (base ** (torch.arange(0, rotary_dim, 2).float() / rotary_dim))
        self.register_buffer("inv_freq", inv_freq)
        self.dim = dim
        self.base = base
        self.interleaved = bool(interleaved)
        self.scaling = _checked_scaling(scaling)
        self.general = rotary_dim != dim or self.interleaved or self.scaling is not None  # (turned without tables, by rotate)
        self._before = []
        self._host_stretch, self._factor = _stretch(rotary_dim // 2, base, self.scaling, "cpu")
        self._settle()
        self.max_seq_len_cached = None
        self.cos_half = None
        self.sin_half = None
        self._captured = []
        self.precision = precision
        self.scale_factor = scale_factor

    def tables(self, seq_len, device):
        """fp32 (cos, sin) half tables [>= seq_len, dim/2] on `device`, built by the HIP table kernel."""
        if self.general:
            raise NotImplementedError("a rotary_dim, interleaved pairs and scaled frequencies have no tables")
        capturing = _capturing(device)
        if self.max_seq_len_cached is None or seq_len > self.max_seq_len_cached or self.cos_half.device != device:
            with torch.inference_mode(False):  # (what an evaluation makes is saved for a backward pass later)
                inv = self.inv_freq.to(device=device, dtype=torch.float32).contiguous()
                tables = K.rope_table(inv, int(seq_len), self.scale_factor)
            if capturing:  # (memory of the graph's, which holds nothing before its first replay)
                return tables
            self.cos_half, self.sin_half = tables
            self.max_seq_len_cached = int(seq_len)
        elif capturing and not any(cos is self.cos_half for cos, _ in self._captured):
            self._captured.append((self.cos_half, self.sin_half))  # (the graph holds no reference to what it reads)
        return self.cos_half, self.sin_half

    def frequencies(self, seq_len, device):
        """(fp64 [rotary_dim / 2] on `device`, the factor of sines and cosines) for a text of seq_len tokens.

        A product of inv_freq and of what its options make of it, computed for every call, on its stream or in its graph: another call, another length, a loaded checkpoint or a moved module
        find nothing of it to replace."""
        stretch = self._stretch if self._stretch.device == device else self._host_stretch.to(device)
        if _goes_by_length(self.scaling):
            stretch = _dynamic_stretch(stretch, self.scaling, seq_len)
        inv_freq = self.inv_freq.to(device)
        inv_freq = inv_freq * stretch if torch.is_tensor(stretch) else inv_freq.double()
        return (inv_freq if self.scale_factor == 1 else inv_freq / self.scale_factor), self._factor

    def _settle(self):
        """The factors of the frequencies go where those are, in 64 bits whatever the module is cast to."""
        device = self.inv_freq.device
        self._stretch = self._host_stretch if device.type in ("cpu", "meta") else self._host_stretch.to(device)

    def _apply(self, fn, *args, **kwargs):
        inv_freq, stretch = self.inv_freq, self._stretch
        super()._apply(fn, *args, **kwargs)
        if stretch.device != self.inv_freq.device:
            self._settle()
        # (what a captured graph may go on reading: a cast to the type that the weights have leaves them, and with them the graph, as they were)
        self._before += [old for old, new in ((inv_freq, self.inv_freq), (stretch, self._stretch)) if old is not new and old.is_cuda]
        return self

    def rotate(self, q, k, position_ids=None, cu_seqlens=None):
        """q [s, b, nq, d], k [s, b, nk, d] -> turned, whatever the options; position_ids int64 [b, s] or None (the place in the sequence).  cu_seqlens: None, or what says that rows hold
        several documents."""
        if _goes_by_length(self.scaling) and (position_ids is not None or cu_seqlens is not None):
            # One set of frequencies holds for a call.  A row's length is that of none of its documents, which would turn by what else lies in the row, and the largest position is the device's.
            raise ValueError('a dynamic scaling goes by the length of texts that fill their rows: with documents packed in a row, or position ids, it needs a "length"')
        if self.scaling is None and self.scale_factor == 1 and self.inv_freq.dtype is torch.float32 and self.inv_freq.device == q.device:
            inv_freq, factor = self.inv_freq, 1.0  # (widened where it is read)
        else:
            inv_freq, factor = self.frequencies(q.shape[0], q.device)
        return F_.rotary_embed(q, k, inv_freq, position_ids, interleaved=self.interleaved, scale=factor)

    def forward(self, x, seq_dim=1, seq_len=None):
        """Reference-shaped return value: (cos, sin) of shape [seq_len, 1, dim] in `precision`."""
        if seq_len is None:
            seq_len = x.shape[seq_dim]
        c, s = self.tables(seq_len, x.device)
        cos = torch.cat((c[:seq_len], c[:seq_len]), dim=-1)[:, None, :]
        sin = torch.cat((s[:seq_len], s[:seq_len]), dim=-1)[:, None, :]
        if self.precision == torch.bfloat16:
            cos, sin = cos.bfloat16(), sin.bfloat16()
        return cos, sin


def apply_rotary_pos_emb(q, k, cos_half, sin_half, position_ids=None):
    """q [s, b, nq, d], k [s, b, nk, d] -> rotated (q, k); position_ids int64 [b, s] or None
    (positions = sequence index), cf. apply_rotary_pos_emb_torch (:105-122)."""
    return F_.apply_rotary_pair(q, k, cos_half, sin_half, position_ids)
