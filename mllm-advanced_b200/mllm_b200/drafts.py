"""Operators that decide on drafted tokens (include/mllmb200_lm.h): logits to probabilities, and verification of drafted tokens
against the target's probabilities from given random numbers.  Calls run on the current stream of the tensors' device, or on
`stream`."""
import torch

from . import lm
from .paged import _fail, _need, _on

_DTYPES = {torch.float32: lm.F32, torch.bfloat16: lm.BF16, torch.float16: lm.F16}


def probabilities(logits, temperature=1.0, out=None, stream=None):
    """Rows of logits [rows, vocab] (fp32, bf16 or fp16) to probabilities in fp32: exp((z - max z) / temperature) over their sum;
    temperature 0: 1 at the first largest.  -inf gives 0, a row of nothing else zeros; NaN or +inf make their row NaN."""
    _need(logits.dim() == 2 and logits.stride(1) == 1 and logits.dtype in _DTYPES and logits.is_cuda, "probabilities: logits [rows, vocab] on the GPU, rows contiguous")
    rows, vocab = logits.shape
    if out is not None:
        _need(out.shape == logits.shape and out.dtype == torch.float32 and out.device == logits.device and out.stride(1) == 1, "probabilities: out like the logits, fp32")

    def call(s):
        o = out if out is not None else torch.empty((rows, vocab), dtype=torch.float32, device=logits.device)
        return lm.lib().mllmb200_lm_probabilities(logits.data_ptr(), _DTYPES[logits.dtype], logits.stride(0), rows, vocab, temperature, o.data_ptr(), max(o.stride(0), vocab), s), o
    st, o = _on(logits.device, stream, call)
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
    _need(target.dim() == 3 and draft.dim() == 3 and target.dtype == draft.dtype == torch.float32, "verify: probabilities [sequences, places, vocab] in fp32")
    seqs, places, vocab = target.shape
    k = places - 1
    _need(k >= 0 and draft.shape == (seqs, k, vocab) and tokens.shape == (seqs, k) and accept.shape == (seqs, k) and pick.shape == (seqs,), "verify: one place more in the target's probabilities than drafts")
    _need(tokens.dtype == torch.int32 and accept.dtype == pick.dtype == torch.float32, "verify: tokens in int32, random numbers in fp32")
    _need(target.stride(2) == 1 and (not k or (draft.stride(2) == 1 and (k == 1 or (tokens.stride(1) == 1 and accept.stride(1) == 1)))) and (seqs < 2 or pick.stride(0) == 1), "verify: rows are contiguous")
    device = target.device
    _need(device.type == "cuda" and all(t.device == device for t in (draft, tokens, accept, pick)), "verify: tensors on one GPU")

    def call(s):
        accepted, out = torch.empty(seqs, dtype=torch.int32, device=device), torch.empty((seqs, places), dtype=torch.int32, device=device)
        st = lm.lib().mllmb200_lm_verify(target.data_ptr(), target.stride(0), target.stride(1), draft.data_ptr(), draft.stride(0), draft.stride(1), tokens.data_ptr(),
                                         tokens.stride(0), accept.data_ptr(), accept.stride(0), pick.data_ptr(), seqs, k, vocab, accepted.data_ptr(), out.data_ptr(), places, s)
        return st, (accepted, out)
    st, o = _on(device, stream, call)
    if st:
        _fail("verify", st)
    return o
