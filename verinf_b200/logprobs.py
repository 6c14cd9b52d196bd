"""What a model's logits say about the tokens that were answered: the log probability of each given token (its negative, in
bits, is the information that the model does not explain), the entropy of the distribution, the likeliest alternatives.
"""
from typing import NamedTuple

import torch

from ._lib import LIB, check, current_device, empty_strided, raw_stream
from .int8 import _FLOATS, DTYPE_CODES, matrix

MAX_TOP = 32


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor       # (rows,) fp32
    entropy: torch.Tensor       # (rows,) fp32
    top_logprob: torch.Tensor   # (rows, top) fp32
    top_token: torch.Tensor     # (rows, top) int64


def token_logprobs(logits, tokens, top=0, temperature=1.0):
    """logits (rows, vocab) fp32 / fp16 / bf16, rows any distance apart (a padded vocabulary's leading columns, say); tokens
    (rows,) int64.  With p = softmax(logits / temperature), natural logarithms throughout:

      logprob      log p of the row's token; 0 for a negative token (a position without one); NaN for a token >= vocab
      entropy      -sum p log p
      top_logprob, top_token   the `top` (0 .. 32) likeliest tokens in falling order, ties to the lowest index

    An entry of -inf is a token that is not allowed; a list with fewer allowed tokens than `top` ends in -1 and -inf.  A row of
    -inf alone has logprob -inf, entropy 0 and an empty list.  A row with a NaN or +inf has NaN in its numbers and an empty
    list (-1).  The token comes before the row: logprob is 0 for a negative token and NaN for one >= vocab whatever the row holds, so
    look for rows that are not valid in entropy.

    The sums are in fp32, in an order that follows the number of rows in the call, the vocabulary and where a row starts: the same
    call gives the same bits, but a row's numbers in a batch may differ in their last bits from those of the row alone (top_token does
    not).  Returns a TokenLogprobs, which carries no gradient."""
    index = logits.get_device() if isinstance(logits, torch.Tensor) else -1
    if index >= 0 and index != current_device():
        with torch.cuda.device(index):
            return token_logprobs(logits, tokens, top, temperature)
    what = "token_logprobs"
    rows, vocab, stride = matrix(logits, what, "logits", _FLOATS)
    if not isinstance(tokens, torch.Tensor) or tokens.dtype is not torch.int64 or tokens.get_device() != index or \
            tokens.shape != (rows,) or not tokens.is_contiguous():
        raise RuntimeError(f"{what}: tokens must be a contiguous int64 tensor of {rows} tokens on the logits' device")
    if not isinstance(top, int) or not 0 <= top <= MAX_TOP:
        raise RuntimeError(f"{what}: top must be 0 .. {MAX_TOP}")
    temperature = float(temperature)
    if not 1e-6 <= temperature <= 1e6:
        raise RuntimeError(f"{what}: temperature must be between 1e-6 and 1e6")
    logprob = empty_strided((rows,), (1,), torch.float32)
    entropy = empty_strided((rows,), (1,), torch.float32)
    top_logprob = empty_strided((rows, top), (top, 1), torch.float32)
    top_token = empty_strided((rows, top), (top, 1), torch.int64)
    rc = LIB.vi_token_logprobs(logits.data_ptr(), DTYPE_CODES[logits.dtype], rows, vocab, stride, tokens.data_ptr(), top, temperature,
                               logprob.data_ptr(), entropy.data_ptr(), top_logprob.data_ptr(), top_token.data_ptr(),
                               raw_stream(index))
    if rc:
        check(rc)
    return TokenLogprobs(logprob, entropy, top_logprob, top_token)
