"""Sampling from logits: temperature, top-k, top-p and min-p, from given random numbers (``twm_sample``, ``include/twm_serve.h``)."""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib
from ._lib import TwmError, check
from .quantize import _require_cuda, _stream_ptr

_DTYPES = {torch.float32: _lib.TWM_F32, torch.float16: _lib.TWM_F16, torch.bfloat16: _lib.TWM_BF16}


@dataclass
class SamplingParams:
    """How a request's tokens are chosen.  temperature 0: greedily; top_k 0, top_p 1 and min_p 0 leave that cut out."""
    temperature: float = 1.0
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0
    seed: int = 0

    def __post_init__(self):
        if not (math.isfinite(self.temperature) and self.temperature >= 0):
            raise ValueError("temperature must be finite and not negative")
        if self.top_k < 0 or not 0 < self.top_p <= 1 or not 0 <= self.min_p <= 1:
            raise ValueError("top_k must not be negative, top_p in (0, 1] and min_p in [0, 1]")


    def generator(self) -> torch.Generator:
        """Random numbers of a request: the same ones for the same seed, however its tokens are dealt to calls."""
        return torch.Generator().manual_seed(self.seed)


class LoopState:
    """Device memory of a decode loop of one row that samples: its settings, which a captured step reads, and the random numbers of
    its steps."""

    def __init__(self, steps: int, device):
        self._settings = torch.zeros(4, dtype=torch.float32, device=device)
        self.random = torch.zeros(max(steps, 1), dtype=torch.float32, device=device)

    def set(self, params: SamplingParams, random: torch.Tensor, at: int = 0) -> None:
        """On the current stream: the settings of the steps to come, and the numbers of steps at, at + 1, ..."""
        top_k = torch.tensor([min(params.top_k, 1 << 30)], dtype=torch.int32).view(torch.float32)
        self._settings.copy_(torch.cat((torch.tensor([params.temperature, params.top_p, params.min_p]), top_k)))
        self.random[at:at + random.numel()].copy_(random)

    def args(self, logits: torch.Tensor, vocab: int, token: int, step: int, history: torch.Tensor, pos: int, length: int) -> _lib.SampleArgs:
        """The call of a step: f32 logits of one row; token, step, pos and length as addresses."""
        p = self._settings.data_ptr()
        return _lib.SampleArgs(1, vocab, _lib.TWM_F32, logits.data_ptr(), vocab, self.random.data_ptr(), p, p + 12, p + 4, p + 8, token, None, step,
                               self.random.numel(), history.data_ptr(), history.numel(), pos, length)


def _column(name: str, t: Optional[torch.Tensor], dtype: torch.dtype, rows: int, index: int) -> int:
    if t is None:
        return 0
    if t.dtype is not dtype or t.numel() != rows or t.get_device() != index or not t.is_contiguous():
        _require_cuda(t)
        raise TwmError(_lib.TWM_EINVAL, f"sample: {name} must be {dtype} [{rows}] on the logits' device")
    return t.data_ptr()


def sample(logits: torch.Tensor, random: torch.Tensor, tokens: torch.Tensor, *, temperature: Optional[torch.Tensor] = None,
           top_k: Optional[torch.Tensor] = None, top_p: Optional[torch.Tensor] = None, min_p: Optional[torch.Tensor] = None,
           prob: Optional[torch.Tensor] = None, stream: Optional[torch.cuda.Stream] = None, flags: int = 0) -> None:
    """tokens int32 [rows]: one of each row of logits (f32, f16 or bf16 [rows, vocab]), chosen by random f32 [rows] in [0, 1).
    temperature, top_p, min_p f32 [rows] and top_k int32 [rows], None to leave one out (1 for the temperature); prob f32 [rows]
    gets what the kept tokens' distribution gave the token.  ``include/twm_serve.h`` has the definition."""
    index = logits.get_device()
    if index < 0:
        _require_cuda(logits)
    dtype, size, ld = _DTYPES.get(logits.dtype), logits.size(), logits.stride()
    if dtype is None or len(size) != 2 or ld[1] != 1:
        raise TwmError(_lib.TWM_EINVAL, "sample: logits must be a float32, float16 or bfloat16 matrix with contiguous rows")
    (rows, vocab), f32, i32 = size, torch.float32, torch.int32
    if rows == 0:
        return
    if torch._C._cuda_getDevice() != index:
        with torch.cuda.device(index):
            return sample(logits, random, tokens, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p, prob=prob, stream=stream, flags=flags)
    args = _lib.pack_sample_args(rows, vocab, dtype, logits.data_ptr(), ld[0] if rows > 1 else vocab, _column("random", random, f32, rows, index),
                                 _column("temperature", temperature, f32, rows, index), _column("top_k", top_k, i32, rows, index),
                                 _column("top_p", top_p, f32, rows, index), _column("min_p", min_p, f32, rows, index),
                                 _column("tokens", tokens, i32, rows, index), _column("prob", prob, f32, rows, index), 0, 0, 0, 0, 0, 0)
    status = _lib.lib().twm_sample(args, flags, _stream_ptr(stream))
    if status:
        check(status, "twm_sample")
