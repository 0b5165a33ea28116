"""Branching continuations: trees of drafted tokens, which of them the model agrees with, and beam search.

Same call contract as :mod:`ft_b200.extend`: the caller owns every tensor (the workspace of :func:`beam_select` comes from torch's
allocator), kernels are enqueued on torch's current CUDA stream of the tensors' device, and no call synchronises with the
host.  Bad arguments raise ``ValueError`` or ``FastTreeError``; what only the device can see is left out and flagged in the device
status word.  The reference leaves all of this to its host; nothing here has a counterpart in it.
"""
from . import lib as _lib
from .extend import ExtendPlan


def _draft_plan(plan):
    if not isinstance(plan, ExtendPlan) or not plan.info.draft:
        raise ValueError("plan must come from fasttree_extend_preparation(..., draft=True)")
    return plan.table, plan._raw


def draft_tree(parents, plan, positions=None):
    """The trees of a step's drafted tokens enter ``plan``, for every :func:`ft_b200.extend.extend` that follows.

    ``parents`` (int32 or int64, one entry per row of ``q``): the number of the token's parent among its request's tokens, an earlier
    one; -1: a root, which hangs on the cached tokens; -2: padding, which sees the cached tokens alone and has no children (anything
    else is taken for padding and flagged).  ``positions`` (int32 or int64, the same length): becomes cached tokens + depth, as
    :func:`ft_b200.extend.append` wants it; 0 deep are roots and padding.  One launch."""
    rc = _lib.call_module().draft_tree(parents, *_draft_plan(plan), positions)
    if rc != 0:
        _lib.check(rc)


def draft_accept(logits, tokens, parents, plan, accepted, counts, next_tokens, slots=None, kv_entries=None, targets=None):
    """Which drafted tokens the model agrees with, in one launch that reads only the logits it needs.

    A request's token 0 is certain (the newest one that was chosen, a root).  From it on, the first child that holds the token of the
    largest logit (of equal ones the lowest; NaN is passed over) is accepted, as long as there is one; the token that no child held is
    the request's next one.  ``logits`` ``[tokens, vocabulary]``, fp16, bf16 or fp32: row t is the model's after token t (a
    row with nothing above -inf gives token 0); or None, with ``targets`` ``[tokens]`` the model's token behind each (sampled ones, say).
    Tokens are whole numbers from 0 that int32 holds: nothing else is accepted, nor matches a target.  ``tokens``, ``parents``: one entry
    per row of ``q``.
    ``accepted`` (int32 ``[requests, at least the longest draft]``): the accepted tokens' numbers, from 0 on, then -1.  ``counts``
    (int32 ``[requests]``): how many.  ``next_tokens`` (int32 or int64 ``[requests]``; int32 has -1 where it does not hold a target); a
    request without tokens, or whose first is no root, has count 0 and -1.  With ``slots`` (the tokens' pool rows, as
    :func:`ft_b200.extend.append` took them) the request's entries of ``kv_entries`` behind its cached ones become the accepted tokens'
    rows, in path order, and then the others', which the caller may free (a row that int32 does not hold becomes -1 and is flagged): the
    request goes on with cached + count tokens in the cache.  No result may overlap what is read, except that one request's ``slots`` may
    be its entries themselves."""
    rc = _lib.call_module().draft_accept(logits, targets, tokens, parents, *_draft_plan(plan), accepted, counts, next_tokens, slots, kv_entries)
    if rc != 0:
        _lib.check(rc)


def beam_select(logits, scores, out_scores, out_beams, out_tokens):
    """The best continuations of each request's beams: score = ``scores[beam] + logits[beam, token] - log sum exp(logits[beam])``.

    ``logits`` ``[batch, beams, vocabulary]``, fp16, bf16 or fp32, any strides with a contiguous vocabulary; ``scores`` fp32
    ``[batch, beams]``.  Results ``[batch, n]``, best first: ``out_scores`` fp32, ``out_beams`` and ``out_tokens`` int32 or int64; at most 64
    beams and results.  Of equal scores the lowest beam's comes first, then the larger logit, then the lowest token.  Logits of -inf are
    never chosen (banned tokens), nor is anything from a beam whose score is not finite (-inf: a beam that ended, or has not begun) or whose
    logits hold NaN or +inf; where too little is left the last results are score -inf, beam -1, token -1.  Logits and scores may be of any
    finite size: tokens masked with the type's lowest value come last, and a score that fp32 does not hold rounds to -inf.  The logarithms
    come from fp32 sums, within 2^-17 up to 131072 logits a row (3e-7 as measured): scores of different beams that are closer may come in
    either order.  ``out_scores`` may be ``scores``, or start with it
    in every row; otherwise no result may overlap what is read.  Two launches."""
    rc = _lib.call_module().beam_select(logits, scores, out_scores, out_beams, out_tokens)
    if rc != 0:
        _lib.check(rc)


def beam_reorder(table, rows, beams, starts=None, ends=None, out_rows=None):
    """Rows of ``table`` follow the beams: columns ``starts[i]`` to ``ends[i]`` (all without) of row ``out_rows[i, j]`` (``rows`` without)
    become those that row ``rows[i, beams[i, j]]`` had before the call, so a request's rows may change places.  For the table of pool rows
    (SGLang's ``req_to_token``: what beams share in the cache stays shared, no key or value moves), token histories, and
    whatever else goes by request.

    ``table`` ``[rows, width]`` of 4- or 8-byte elements; ``rows`` ``[batch, beams]``, ``beams`` and ``out_rows`` ``[batch, n]`` (int32 or
    int64, at most 64 each); beam -1 leaves its row alone.  A row that is written belongs to one request and stands once among its
    ``out_rows``.  The table must not overlap the numbers.  One launch."""
    rc = _lib.call_module().beam_reorder(table, rows, beams, out_rows, starts, ends)
    if rc != 0:
        _lib.check(rc)
