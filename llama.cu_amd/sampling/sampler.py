"""Sampling on the device from rows of float32 logits (kernels: csrc/kernels/sampling.hip).

The uniform number of a draw comes from a counter-based generator keyed by the
request's seed, its id and the index of the token it draws: a request's tokens do not
depend on what else is in the batch or on how its prompt was cut.
"""
from __future__ import annotations

import array
import ctypes
import functools
from typing import List, Optional, Sequence, Tuple, Union

import torch

from ..kernels import build, ops
from ..kernels.ops import KernelError, _check, _gpu, _ptr, _stream, to_device as _to_device
from .params import SamplingParams

_MASK = (1 << 64) - 1
MAX_VOCAB = 1 << 19          # what the kernels' 64-bit sums of weights allow
MAX_DRAFTS = 1024            # drafts a request in one verification


def _splitmix64(x: int) -> int:
    x = (x + 0x9E3779B97F4A7C15) & _MASK
    z = x
    z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & _MASK
    z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & _MASK
    return z ^ (z >> 31)


# what a number is drawn for: a token; whether a draft stands; the token after the drafts that do
DRAW, JUDGE, FINAL = 0, 1, 2


def uniform(seed: int, request: int, index: int, purpose: int = DRAW) -> float:
    """A number in [0, 1) with 24 random bits, a pure function of its keys."""
    h = _splitmix64(seed & _MASK)
    if purpose:
        h = _splitmix64(h ^ purpose)
    h = _splitmix64(h ^ (request & _MASK))
    h = _splitmix64(h ^ (index & _MASK))
    return (h >> 40) / float(1 << 24)


def argmax(logits: torch.Tensor) -> torch.Tensor:
    """The index of the largest logit of each row (the lowest among equals), int32."""
    _gpu(logits)
    if logits.dim() != 2 or logits.dtype != torch.float32 or logits.stride(1) != 1:
        raise KernelError("argmax: logits must be float32 [rows, vocab] with contiguous rows")
    rows, vocab = logits.shape
    out = torch.empty(rows, dtype=torch.int32, device=logits.device)
    # a long row is read by several workgroups, whose winners a second kernel compares
    parts = max(1, min(16, vocab // 8192))
    part_val = torch.empty(rows * parts, dtype=torch.float32, device=logits.device) if parts > 1 else None
    part_idx = torch.empty(rows * parts, dtype=torch.int32, device=logits.device) if parts > 1 else None
    lib = build.load("sampling")
    _check(lib.lcu_argmax(_ptr(logits), logits.stride(0), rows, vocab, _ptr(out), parts, _ptr(part_val), _ptr(part_idx),
                          _stream()), "argmax")
    return out


def sample_rows(logits: torch.Tensor, temperature: Sequence[float], top_p: Sequence[float], top_k: Sequence[int],
                u: Sequence[float]) -> torch.Tensor:
    """One draw per row with the row's temperature (> 0), top_p, top_k and uniform number."""
    _gpu(logits)
    if logits.dim() != 2 or logits.dtype != torch.float32 or logits.stride(1) != 1:
        raise KernelError("sample: logits must be float32 [rows, vocab] with contiguous rows")
    rows, vocab = logits.shape
    if not (len(temperature) == len(top_p) == len(top_k) == len(u) == rows):
        raise KernelError("sample: one temperature, top_p, top_k and uniform number per row")
    if any(not t > 0 for t in temperature) or any(not 0 <= x < 1 for x in u):
        raise KernelError("sample: temperatures must be > 0 and uniform numbers in [0, 1)")
    dev = logits.device
    fl = _to_device([list(temperature), list(top_p), list(u)], torch.float32, dev)
    kk = _to_device([min(int(k), vocab) for k in top_k], torch.int32, dev)
    out = torch.empty(rows, dtype=torch.int32, device=dev)
    lib = build.load("sampling")
    # a long row is cut into parts, one workgroup each: about one workgroup per compute unit in all
    parts = max(1, min(16, 256 // rows, vocab // 4096))
    lib.lcu_sample_scratch_bytes.restype = ctypes.c_size_t
    scratch = torch.zeros(int(lib.lcu_sample_scratch_bytes(rows, parts)), dtype=torch.uint8, device=dev)
    any_top_k = any(int(k) < vocab for k in top_k)
    _check(lib.lcu_sample(_ptr(logits), logits.stride(0), rows, vocab, _ptr(fl[0]), _ptr(fl[1]), _ptr(kk), _ptr(fl[2]),
                          _ptr(out), int(any_top_k), parts, _ptr(scratch), _stream()), "sample")
    return out


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor) -> torch.Tensor:
    """``log softmax(logits[r])[tokens[r]]`` for every row: the natural logarithm of the probability that the model
    gives each row's token (float32, on the device).  The reference hands back the chosen token's value beside its
    index (``KVPair``, llama.cu/src/op/random_sample/mod.rs:29-36); this is that value made comparable across rows."""
    _gpu(logits, tokens)
    if logits.dim() != 2 or logits.dtype != torch.float32 or logits.stride(1) != 1:
        raise KernelError("token_logprobs: logits must be float32 [rows, vocab] with contiguous rows")
    rows, vocab = logits.shape
    if tokens.dtype != torch.int32 or tokens.numel() != rows or not tokens.is_contiguous():
        raise KernelError(f"token_logprobs: tokens must be a contiguous int32 tensor of {rows} entries")
    out = torch.empty(rows, dtype=torch.float32, device=logits.device)
    lib = build.load("sampling")
    _check(lib.lcu_token_logprob(_ptr(logits), logits.stride(0), rows, vocab, _ptr(tokens), _ptr(out), _stream()), "token_logprobs")
    return out


def _options(values, dtype: torch.dtype, rows: int, device, what: str, fine, why: str):
    """A number a row, and the least of them: a sequence, which is looked at here, or a tensor that is on the device already, which is not (its least: None)."""
    if isinstance(values, torch.Tensor) and values.is_cuda:
        if values.device != device or values.dtype != dtype or values.shape != (rows,) or not values.is_contiguous():
            raise KernelError(f"token_probs: {what} on the device must be contiguous {dtype} [{rows}], got {values.dtype} {tuple(values.shape)}")
        return values, None
    values = values.tolist() if isinstance(values, torch.Tensor) else list(values)
    low = min(values, default=1)
    total = sum(values)                # (in which a NaN shows)
    if len(values) != rows or (rows and not (total == total and fine(low, values))):
        raise KernelError(f"token_probs: {what} must be {rows} numbers {why}")
    return values, low


def _packed(kind: str, values, most: int):
    """A sequence's numbers as the kernels have them; counts that no 32 bits hold are the vocabulary's."""
    if kind == "i":
        try:
            return array.array("i", values)
        except (OverflowError, TypeError):
            values = [int(k) if k < most else most for k in values]
    return array.array(kind, values)


@functools.lru_cache(maxsize=1024)
def _probs_scratch(rows: int, vocab: int, parts: int, cuts: bool) -> int:
    size = build.load("token_probs").lcu_token_probs_scratch_bytes
    size.restype = ctypes.c_size_t
    return size(rows, vocab, parts, int(cuts))


def token_probs(logits: torch.Tensor, temperature, top_p, top_k, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The distribution that ``sample_rows`` draws each row's token from, float32 ``[rows, vocab]``: with the logits in descending order
    (equal ones by index), weights ``w_i = exp((l_i - l_0) / T)`` and sums ``c`` of them, entry ``i`` has the share
    ``(min(c_i, L) - min(c_{i-1}, L)) / L``, ``L = min(top_p * c_n, c_{top_k})``.  A temperature of 0, or ``top_k`` 1, leaves the first
    of the largest logits.  A NaN counts as -inf, which has no share; a row of nothing else is all zeros.

    ``temperature``, ``top_p``, ``top_k``: a sequence of one number a row, or (float32, float32, int32) tensors on the logits' device,
    whose numbers are not looked at: a temperature or top_p that is not positive, or a top_k below 1, then acts as a temperature of 0.
    A call of more than 64 rows that is captured into a graph takes tensors."""
    if logits.dim() != 2 or logits.dtype != torch.float32 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise KernelError("token_probs: logits must be float32 [rows, vocab] with contiguous rows")
    rows, vocab = logits.shape
    if not 0 < vocab <= MAX_VOCAB:
        raise KernelError(f"token_probs: a vocabulary of {vocab} is not supported (1 to {MAX_VOCAB})")
    dev = logits.device
    temperature, _ = _options(temperature, torch.float32, rows, dev, "temperature", lambda low, v: low >= 0 and max(v) < float("inf"), ">= 0")
    top_p, least_p = _options(top_p, torch.float32, rows, dev, "top_p", lambda low, _: low > 0, "> 0")
    top_k, least_k = _options(top_k, torch.int32, rows, dev, "top_k", lambda low, _: low >= 1, ">= 1")
    if out is None:
        out = torch.empty_strided((rows, vocab), (vocab, 1), dtype=torch.float32, device=dev)
    else:
        if out.shape != (rows, vocab) or out.dtype != torch.float32 or not out.is_contiguous():
            raise KernelError(f"token_probs out: must be contiguous float32 {(rows, vocab)}, got {out.dtype} {tuple(out.shape)}")
        ops.apart("token_probs", out, logits, *[v for v in (temperature, top_p, top_k) if isinstance(v, torch.Tensor)])
    ops.here("token_probs", logits, out)
    if rows == 0:
        return out
    # whether some row is cut: known of sequences, taken as given of tensors
    cuts = least_p is None or least_k is None or least_p < 1 or least_k < vocab
    sequences = [None if isinstance(v, torch.Tensor) else _packed("f" if i < 2 else "i", v, vocab) for i, v in enumerate((temperature, top_p, top_k))]
    at = [v.data_ptr() if isinstance(v, torch.Tensor) else None for v in (temperature, top_p, top_k)]
    given = None
    if any(v is not None for v in sequences):
        data = bytearray(b"".join(v.tobytes() for v in sequences if v is not None))
        if rows <= 64 and all(v is not None for v in sequences):
            given = (ctypes.c_char * len(data)).from_buffer(data)             # in the launch itself
        else:
            if torch.cuda.is_current_stream_capturing():
                raise KernelError("token_probs: a captured call of more than 64 rows, or with some options as tensors, takes all of them as tensors on the device "
                                  "(a replay would read a sequence's memory again, which is gone by then)")
            host = torch.empty(len(data), dtype=torch.uint8, pin_memory=True)
            host.copy_(torch.frombuffer(data, dtype=torch.uint8))
            there = host.to(dev, non_blocking=True)
            place = there.data_ptr()
            for i, v in enumerate(sequences):
                if v is not None:
                    at[i], place = place, place + 4 * rows
    # a long row is cut into parts of 4,096 logits at least, one workgroup each, up to about four workgroups a compute unit in all
    parts = max(1, min(32, 4 * ops.TUNING.compute_units // rows, vocab // 4096))
    size = _probs_scratch(rows, vocab, parts, cuts)
    scratch = torch.empty_strided((size,), (1,), dtype=torch.uint8, device=dev) if size else None
    _check(ops.bind("token_probs", "lcu_token_probs", "pliipppppiip")(logits.data_ptr(), logits.stride(0), rows, vocab, *at, given, out.data_ptr(), parts, int(cuts),
                                                                     None if scratch is None else scratch.data_ptr(), ops.raw_stream()), "token_probs")
    return out


def _rows_of(t: torch.Tensor, what: str, vocab: Optional[int] = None, rows: Optional[int] = None) -> None:
    if t.dim() != 2 or t.dtype != torch.float32 or (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]) \
            or vocab not in (None, t.shape[1]) or rows not in (None, t.shape[0]):
        raise KernelError(f"verify_drafts: {what} must be float32 [{'rows' if rows is None else rows}, {'vocab' if vocab is None else vocab}] with contiguous rows, "
                          f"got {t.dtype} {tuple(t.shape)} with strides {t.stride()}")


def verify_drafts(probs: torch.Tensor, starts: torch.Tensor, drafts: torch.Tensor, accept: torch.Tensor, final: torch.Tensor, max_drafts: int,
                  draft_probs: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Which of the requests' drafted tokens stand, and the token after them, so that what comes out is distributed as the target's tokens are.

    ``probs`` (float32 ``[rows, vocab]``): the target's probabilities (``token_probs``), for every request one row more than it has drafts, the
    requests one after the other; request ``b`` has the rows ``starts[b]`` to ``starts[b + 1]`` (int32, one entry more than requests, the first 0).
    ``drafts`` (int32), ``accept`` (float32 in [0, 1)) and ``draft_probs`` (float32 ``[drafts, vocab]``, what the drafts were drawn from; without it
    they were certain) hold all requests' drafts one after the other; ``final`` (float32 in [0, 1)) one number a request.

    Draft ``i`` stands if ``accept * q_i(d_i) < p_i(d_i)``, and the first that does not is the last looked at.  The token after those that stand is the
    first ``v`` whose sum of ``max(p - q, 0)`` up to ``v`` is more than ``final`` times the whole (of ``p`` itself where all stand, and where ``max(p - q,
    0)`` leaves nothing).  Probabilities that are no finite positive numbers count as zero, a draft outside the vocabulary never stands.

    Returns ``(accepted [requests], tokens [requests, max_drafts + 1])``, int32 on the device: a request's drafts that stand, the token after them (-1 if
    its row holds no probability at all), and -1 behind.  A request whose ``starts`` make no sense, or that has more than ``max_drafts`` drafts, gets 0
    and -1 only."""
    _rows_of(probs, "probs")
    rows, vocab = probs.shape
    if starts.dtype != torch.int32 or starts.dim() != 1 or starts.numel() < 1 or not starts.is_contiguous():
        raise KernelError("verify_drafts: starts must be a contiguous int32 [requests + 1]")
    requests = starts.numel() - 1
    n = rows - requests
    if drafts.dtype != torch.int32 or drafts.shape != (n,) or not drafts.is_contiguous():
        raise KernelError(f"verify_drafts: {rows} rows of {requests} requests judge {n} drafts: drafts must be contiguous int32 [{n}], got {drafts.dtype} {tuple(drafts.shape)}")
    for t, what, size in ((accept, "accept", n), (final, "final", requests)):
        if t.dtype != torch.float32 or t.shape != (size,) or not t.is_contiguous():
            raise KernelError(f"verify_drafts: {what} must be contiguous float32 [{size}], got {t.dtype} {tuple(t.shape)}")
    if draft_probs is not None:
        _rows_of(draft_probs, "draft_probs", vocab, n)
    if not 0 <= int(max_drafts) <= MAX_DRAFTS:
        raise KernelError(f"verify_drafts: max_drafts {max_drafts} is not supported (0 to {MAX_DRAFTS})")
    if not 0 < vocab <= MAX_VOCAB:
        raise KernelError(f"verify_drafts: a vocabulary of {vocab} is not supported (1 to {MAX_VOCAB})")
    ops.here("verify_drafts", probs, starts, drafts, accept, final, draft_probs)
    dev, width = probs.device, int(max_drafts) + 1
    accepted = torch.empty_strided((requests,), (1,), dtype=torch.int32, device=dev)
    tokens = torch.empty_strided((requests, width), (width, 1), dtype=torch.int32, device=dev)
    if requests == 0:
        return accepted, tokens
    # the row at which a run ends is cut into parts of 2,048 tokens, one workgroup each: what a workgroup of the second launch takes at once; a workgroup a request does all of a short one
    parts = 1 if vocab <= 8192 else min(64, -(-vocab // 2048))
    sums = torch.empty_strided((requests * parts * 2,), (1,), dtype=torch.float64, device=dev) if parts > 1 else None
    _check(ops.bind("verify", "lcu_verify_drafts", "plipipiplppiiippp")(
        probs.data_ptr(), probs.stride(0), rows, starts.data_ptr(), requests, drafts.data_ptr() if n else None, n, None if draft_probs is None else draft_probs.data_ptr(),
        0 if draft_probs is None else draft_probs.stride(0), accept.data_ptr() if n else None, final.data_ptr(), vocab, int(max_drafts), parts, None if sums is None else sums.data_ptr(), accepted.data_ptr(),
        tokens.data_ptr(), ops.raw_stream()), "verify_drafts")
    return accepted, tokens


class Sampler:
    def probs(self, logits: torch.Tensor, params: Sequence[SamplingParams]) -> torch.Tensor:
        """Every row's distribution under its options (``token_probs``): what ``sample_device`` draws the row's token from."""
        if len(params) != logits.shape[0]:
            raise KernelError(f"probs: {logits.shape[0]} rows with options for {len(params)}")
        return token_probs(logits, [0.0 if p.is_argmax else p.temperature for p in params], [p.top_p for p in params], [p.top_k for p in params])

    def verify(self, logits: torch.Tensor, drafts: Sequence[Sequence[int]], params: Sequence[SamplingParams], keys: Sequence[Tuple[int, int]],
               draft_probs: Optional[torch.Tensor] = None) -> List[List[int]]:
        """The tokens that drafted ones turn into: of request ``i`` its drafts that stand and the token after them, distributed as tokens drawn one
        after the other from the model's own logits.  ``logits`` (float32): for every request a row for each of its drafts and one more, the
        requests one after the other; ``draft_probs``: what the drafts were drawn from, a row each (``probs`` of the drafting model's logits;
        None: they were certain, found in the text or greedy); ``keys[i] = (request id, index of its first drafted token)``.  Whether drafts stand
        is judged by numbers of their own, not by those that ``sample`` draws tokens with."""
        if not (len(drafts) == len(params) == len(keys)):
            raise KernelError("verify: drafts, options and keys, one of each a request")
        counts = [len(d) for d in drafts]
        if logits.dim() != 2 or logits.shape[0] != sum(counts) + len(drafts):
            raise KernelError(f"verify: {sum(counts)} drafts of {len(drafts)} requests need {sum(counts) + len(drafts)} rows of logits, got {tuple(logits.shape)}")
        if not drafts:
            return []
        probs = self.probs(logits, [p for p, c in zip(params, counts) for _ in range(c + 1)])
        starts, flat, judge, final = [0], [], [], []
        for d, p, (request, index) in zip(drafts, params, keys):
            starts.append(starts[-1] + len(d) + 1)
            flat += [int(t) for t in d]
            judge += [uniform(p.seed, request, index + j, JUDGE) for j in range(len(d))]
            final.append(uniform(p.seed, request, index, FINAL))
        dev = logits.device
        ints, floats = _to_device(starts + flat, torch.int32, dev), _to_device(judge + final, torch.float32, dev)
        accepted, tokens = verify_drafts(probs, ints[:len(starts)], ints[len(starts):], floats[:len(flat)], floats[len(flat):], max(counts), draft_probs)
        both = torch.cat([accepted.unsqueeze(1), tokens], dim=1).tolist()
        return [row[1:row[0] + 2] for row in both]

    def sample_device(self, logits: torch.Tensor, params: Sequence[SamplingParams],
                      keys: Sequence[Tuple[int, int]]) -> torch.Tensor:
        """A token for every row, left on the device (int32)."""
        random_rows = [i for i, p in enumerate(params) if not p.is_argmax]
        if random_rows and len(random_rows) == logits.shape[0]:
            return sample_rows(logits, [p.temperature for p in params], [p.top_p for p in params], [p.top_k for p in params],
                               [uniform(p.seed, k[0], k[1]) for p, k in zip(params, keys)])
        out = argmax(logits)
        if random_rows:
            # the rows that draw are gathered, drawn from and put back by the engine's own small kernels
            both = _to_device([random_rows, list(range(len(random_rows)))], torch.int32, logits.device)
            sub = ops.gather_rows(logits, both[0])
            drawn = sample_rows(sub, [params[i].temperature for i in random_rows], [params[i].top_p for i in random_rows],
                                [params[i].top_k for i in random_rows],
                                [uniform(params[i].seed, keys[i][0], keys[i][1]) for i in random_rows])
            ops.feed_tokens(out, drawn, both[1], both[0])               # out[random_rows[i]] = drawn[i]
        return out

    def sample(self, logits: torch.Tensor, params: Sequence[SamplingParams],
               keys: Sequence[Tuple[int, int]]) -> List[int]:
        """A token for every row.  ``keys[i] = (request id, index of the drawn token)``."""
        rows = logits.shape[0]
        if rows == 0:
            return []
        greedy = argmax(logits)
        random_rows = [i for i, p in enumerate(params) if not p.is_argmax]
        if not random_rows:
            return greedy.tolist()
        sub = logits if len(random_rows) == rows else ops.gather_rows(logits, _to_device(random_rows, torch.int32, logits.device))
        drawn = sample_rows(sub, [params[i].temperature for i in random_rows], [params[i].top_p for i in random_rows],
                            [params[i].top_k for i in random_rows],
                            [uniform(params[i].seed, keys[i][0], keys[i][1]) for i in random_rows]).tolist()
        out = greedy.tolist()
        for i, t in zip(random_rows, drawn):
            out[i] = t
        return out
