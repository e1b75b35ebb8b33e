"""Operators that decide on drafted tokens (include/mllmb200_lm.h): logits to probabilities, and verification of drafted tokens
against the target's probabilities from given random numbers.  Calls run on the current stream of the tensors' device, or on
`stream`."""
import torch

from . import lm
from .paged import _fail, _on, _refuse

_DTYPES = {torch.float32: lm.F32, torch.bfloat16: lm.BF16, torch.float16: lm.F16}


def probabilities(logits, temperature=1.0, out=None, stream=None):
    """Rows of logits [rows, vocab] (fp32, bf16 or fp16) to probabilities in fp32: exp((z - max z) / temperature) over their sum;
    temperature 0: 1 at the first largest.  -inf gives 0, a row of nothing else zeros; NaN or +inf make their row NaN."""
    dtype = _DTYPES.get(logits.dtype)
    distance = None if out is None or logits.dim() != 2 else lm.row_distance("probabilities", out, *logits.shape)
    if not (logits.dim() == 2 and (logits.shape[1] < 2 or logits.stride(1) == 1) and dtype is not None and logits.is_cuda):
        _refuse("probabilities", (lambda: False, "logits [rows, vocab] in fp32, bf16 or fp16 on the GPU, rows contiguous"))
    rows, vocab = logits.shape
    if out is not None and out.get_device() != logits.get_device():
        _refuse("probabilities", (lambda: False, "out on the logits' GPU"))

    def call(s):
        o = out if out is not None else logits.new_empty((rows, vocab), dtype=torch.float32)
        return lm.lib().mllmb200_lm_probabilities(logits.data_ptr(), dtype, logits.stride(0), rows, vocab, temperature, o.data_ptr(), distance or vocab, s), o
    st, o = _on(logits.get_device(), stream, call, logits, out)
    if st:
        _fail("probabilities", st)
    return o


def verify(target, draft, tokens, accept, pick, stream=None):
    """Which drafted tokens stand, and the token behind them, so that what comes out is distributed as the target's own draws.

    target: fp32 [sequences, drafts + 1, vocab], the target's probabilities behind every place; draft: fp32 [sequences, drafts,
    vocab], those that tokens (int32 [sequences, drafts]) were drawn from; accept: fp32 [sequences, drafts] and pick: fp32
    [sequences], uniform in [0, 1).  Token x at place i is accepted while accept * draft(x) < target(x).  At the first refused
    place the next token comes from max(target - draft, 0), behind the last draft from the target: the lowest index whose
    running sum exceeds pick times the whole.  A token outside of the vocabulary ends a sequence's drafts.  No drafts: a draw.

    Returns accepted (int32 [sequences]) and the new tokens (int32 [sequences, drafts + 1]): the accepted ones, the next
    one, -1 behind it."""
    try:
        seqs, places, vocab = target.shape
        d_seq, d_row, d_one = draft.stride()
        tokens_seq, tokens_one = tokens.stride()
        accept_seq, accept_one = accept.stride()
    except ValueError:
        _refuse("verify", (lambda: False, "probabilities [sequences, places, vocab], tokens and random numbers [sequences, drafts]"))
    k, device = places - 1, target.get_device()
    t_seq, t_row, t_one = target.stride()
    if not (k >= 0 and draft.shape == (seqs, k, vocab) and tokens.shape == (seqs, k) and accept.shape == (seqs, k) and pick.shape == (seqs,) and
            target.dtype == draft.dtype == accept.dtype == pick.dtype == torch.float32 and tokens.dtype == torch.int32 and (vocab < 2 or (t_one == 1 and (k == 0 or d_one == 1))) and
            (k < 2 or (tokens_one == 1 and accept_one == 1)) and (seqs < 2 or pick.stride(0) == 1) and device >= 0 and
            draft.get_device() == tokens.get_device() == accept.get_device() == pick.get_device() == device):
        _refuse("verify", (lambda: k >= 0 and draft.shape == (seqs, k, vocab) and tokens.shape == accept.shape == (seqs, k) and pick.shape == (seqs,), "one place more in the target's probabilities than drafts"),
                (lambda: target.dtype == draft.dtype == accept.dtype == pick.dtype == torch.float32 and tokens.dtype == torch.int32, "tokens in int32, all else in fp32"),
                (lambda: device >= 0 and all(t.get_device() == device for t in (draft, tokens, accept, pick)), "tensors on one GPU"), (lambda: False, "rows are contiguous"))

    def call(s):
        accepted, out = torch.empty_like(pick, dtype=torch.int32), tokens.new_empty((seqs, places))
        st = lm.lib().mllmb200_lm_verify(target.data_ptr(), t_seq, t_row, draft.data_ptr(), d_seq, d_row, tokens.data_ptr(), tokens_seq, accept.data_ptr(), accept_seq,
                                         pick.data_ptr(), seqs, k, vocab, accepted.data_ptr(), out.data_ptr(), places, s)
        return st, (accepted, out)
    st, o = _on(device, stream, call, target, draft, tokens, accept, pick)
    if st:
        _fail("verify", st)
    return o
