"""New tokens of a serving step: into the paged cache (``append``) and their attention over it (``extend``).

Same call contract as :mod:`ft_b200.engine`: the caller owns every tensor, kernels are enqueued on torch's current CUDA
stream of the tensors' device, and ``append`` and ``extend`` do not synchronise with the host.  ``prepare``, once per step, does: it
copies the plan from ordinary host memory and returns when the copy is done.  Bad arguments raise ``ValueError`` or
``FastTreeError``.  The reference leaves both to its host (SGLang's rotary embedding, ``store_kv_cache`` and extend
attention); they have no counterpart in it.
"""
import ctypes

import numpy as np
import torch

from . import lib as _lib


def append(q, k, v, k_buffer, v_buffer, slots, q_out=None, positions=None, cos_sin=None, sections=None, interleaved=False):
    """Turn ``q`` and ``k`` by their tokens' positions and write ``k`` / ``v`` to the pool rows ``slots``, in one launch.

    ``q`` ``[tokens, q heads, head_dim]`` (or None), ``k`` and ``v`` ``[tokens, kv heads, head_dim]``, the pool
    ``[rows, kv heads, head_dim]``; fp16, bf16 or fp32, any strides with a contiguous head_dim axis.  ``slots`` (int32 or
    int64): -1 is a padding token, which is not stored; no row twice.  ``k`` and ``v`` may be views of the pool only where each
    token stands at its own slot.  The turned queries go to ``q_out``, which may be ``q``
    (the default) but must not overlap it, ``k``, ``v`` or the pool otherwise.  ``cos_sin`` (fp32 ``[positions,
    rot_dim]``): cosines of the rot_dim / 2 pairs, then their sines; elements from ``rot_dim`` on stay as they are.
    ``positions``: ``[tokens]``, or ``[axes, tokens]`` with ``sections``, the number of consecutive pairs that each axis turns.
    Pairs are elements (i, i + rot_dim / 2), or (2 i, 2 i + 1) if ``interleaved``.  Without ``positions`` and ``cos_sin``
    nothing is turned (``q``, if given, is copied to ``q_out``)."""
    rc = _lib.call_module().append(q, k, v, k_buffer, v_buffer, slots, q_out, positions, cos_sin, sections, interleaved)
    if rc != 0:
        _lib.check(rc)


class ExtendPlan:
    """Schedule of one step's extend attention, for all layers: a host description and one device table.  Read-only once
    made: any number of calls, streams and captured graphs may use it at once.  Like every tensor of a call, its table has to
    live until the work that reads it is done: keep the plan as long as a graph that was captured with it, and until other
    streams than the one it was made on are through with it.  A plan is of one step's lengths, and so is a graph that was
    captured with it."""

    def __init__(self, info, table, seq_lens, extend_lens):
        self.info = info
        self.table = table
        self.seq_lens, self.extend_lens = seq_lens, extend_lens
        self._raw = bytes(info)

    @property
    def num_tokens(self):
        return int(self.info.num_tokens)

    @property
    def partial_rows(self):
        return int(self.info.partial_rows)


def _ints(name, x, n=None):
    if isinstance(x, torch.Tensor):
        if x.is_cuda:
            raise ValueError(f"{name} must be on the host: the plan is made there")
        x = x.numpy()
    a = np.asarray(x)
    if a.size and not np.issubdtype(a.dtype, np.integer):
        raise ValueError(f"{name} must be integers")
    a = np.ascontiguousarray(a.astype(np.int64)).reshape(-1)
    if n is not None and a.size != n:
        raise ValueError(f"{name} must have one entry per request ({n}), got {a.size}")
    return a


def _order_by_prefix(n, cached, shared_prefixes):
    """Order of the requests in which those that share stand together, and how many leading tokens each is known to share
    with the one before it."""
    of = [[] for _ in range(n)]
    groups = []
    for members, length in shared_prefixes:
        members, length = [int(m) for m in members], int(length)
        if length < 0:
            raise ValueError("a shared prefix has a negative length")
        for m in members:
            if not 0 <= m < n:
                raise ValueError(f"a shared prefix names request {m} of {n}")
            if length > cached[m]:
                raise ValueError(f"a shared prefix of {length} tokens is longer than the {int(cached[m])} cached ones of request {m}")
        if length and len(set(members)) > 1:
            groups.append((length, -len(set(members)), len(groups), set(members)))
    groups.sort(key=lambda g: g[:3])
    for i, g in enumerate(groups):
        for m in g[3]:
            of[m].append(i)
    order = sorted(range(n), key=lambda r: (of[r] == [], of[r], r))
    shared = np.zeros(n, dtype=np.int64)
    for a in range(1, n):
        both = set(of[order[a - 1]]).intersection(of[order[a]])
        shared[a] = max((groups[i][0] for i in both), default=0)
    return order, shared


def host_plan(seq_lens, extend_lens, kv_starts, num_qo_heads, num_kv_heads, head_dim, dtype, shared_prefixes=None, window=0,
              num_sms=148, draft=False):
    """Host half of :func:`prepare`: ``(info, numpy int32 table, seq_lens, extend_lens)``."""
    seq = _ints("seq_lens", seq_lens)
    n = seq.size
    ext, start = _ints("extend_lens", extend_lens, n), _ints("kv_starts", kv_starts, n)
    if dtype not in (torch.float16, torch.bfloat16, torch.float32):
        raise ValueError(f"unsupported dtype {dtype}")
    if n and (ext.min() < 0 or (seq - ext).min() < 0):
        raise ValueError("extend_lens must lie between 0 and seq_lens")
    if n and start.min() < 0:
        raise ValueError("kv_starts must not be negative")
    if int(window) < 0:
        raise ValueError("window must not be negative")
    if num_qo_heads <= 0 or num_kv_heads <= 0 or num_qo_heads % num_kv_heads:
        raise ValueError(f"num_qo_heads {num_qo_heads} must be a multiple of num_kv_heads {num_kv_heads}")
    q_start = np.concatenate([[0], np.cumsum(ext)[:-1]]).astype(np.int64) if n else np.zeros(0, dtype=np.int64)
    order, shared = _order_by_prefix(n, seq - ext, shared_prefixes or [])
    arrays = [np.ascontiguousarray(a[order]) if n else a for a in (seq, ext, start, q_start)] + [shared]
    lib = _lib.load()
    i64p, handle = ctypes.POINTER(ctypes.c_int64), ctypes.c_void_p()
    sizes = (n, int(num_qo_heads), int(num_kv_heads), int(head_dim), 4 if dtype == torch.float32 else 2, min(int(window), 2 ** 31 - 1),
             int(num_sms), ctypes.byref(handle))
    if draft:
        if n and ext.max() > _lib.FT_MAX_DRAFT:
            raise ValueError(f"a request has {int(ext.max())} drafted tokens, more than {_lib.FT_MAX_DRAFT}")
        ids = np.asarray(order, dtype=np.int32)
        rc = lib.ft_draft_plan_build(*(a.ctypes.data_as(i64p) for a in arrays), ids.ctypes.data_as(ctypes.POINTER(ctypes.c_int32)), *sizes)
    else:
        rc = lib.ft_extend_plan_build(*(a.ctypes.data_as(i64p) for a in arrays), *sizes)
    if rc != 0:
        raise _lib.FastTreeError(rc, "ft_extend_plan_build refused the step: head_dim must be one of 16, 32, 64, 128, 256 and the "
                                     "step's tables must fit 32-bit fields")
    try:
        info = _lib.ExtendPlanInfo()
        _lib.check(lib.ft_extend_plan_get_info(handle, ctypes.byref(info)))
        table = np.zeros(max(4, int(info.table_ints)), dtype=np.int32)
        _lib.check(lib.ft_extend_plan_copy(handle, table.ctypes.data_as(ctypes.POINTER(ctypes.c_int32))))
    finally:
        lib.ft_extend_plan_free(handle)
    return info, table, seq.tolist(), ext.tolist()


def prepare(seq_lens, extend_lens, kv_starts, num_qo_heads, num_kv_heads, head_dim, dtype, shared_prefixes=None, window=0,
            device="cuda", draft=False):
    """Plan a step's extend attention; the plan serves every layer of the step.

    Request r has ``seq_lens[r]`` tokens in the cache, the last ``extend_lens[r]`` of them the step's new ones, whose
    queries are the next rows of ``q`` (requests in order).  The pool rows of its tokens are ``kv_entries[kv_starts[r]:]``
    (in SGLang: row ``req_pool_indices[r]`` of ``req_to_token``, flattened).  ``shared_prefixes``: pairs ``(requests,
    length)`` - these requests' first ``length`` cached tokens are the same pool rows, and their attention reads them once;
    nested pairs describe a tree (:func:`tree_prefixes`).  ``window`` > 0: a token sees the newest ``window`` positions up
    to its own.  Integers on the host; one copy to ``device``, for which the host waits.  Steps of single tokens without window
    and cap are ``fasttree_decode``'s: it takes them faster and without a plan per step.

    ``draft``: a request's new tokens are the nodes of a tree (at most 1024, parents first), not a chain: a token sees the cached
    tokens, its ancestors and itself; with a window those of the newest ``window`` positions up to its own, which is cached + depth.
    The plan goes by the sizes; the trees, which may live on the device alone, are given to :func:`ft_b200.branch.draft_tree` before
    the step's first :func:`extend` (until then tokens are chains).  That changes the plan's table, so such a plan belongs to one
    stream, or the caller orders what uses it."""
    dev = torch.device(device)
    if dev.type != "cuda":
        raise ValueError("the plan is uploaded to a CUDA device; the engine has no CPU path")
    sms = torch.cuda.get_device_properties(dev).multi_processor_count
    info, table, seq, ext = host_plan(seq_lens, extend_lens, kv_starts, num_qo_heads, num_kv_heads, head_dim, dtype,
                                      shared_prefixes, window, sms, draft)
    return ExtendPlan(info, torch.from_numpy(table).to(dev), seq, ext)


def tree_prefixes(tree_info):
    """``shared_prefixes`` of a tree of ``KVTreeNode`` records whose nodes are the requests' cached prefixes."""
    depth, out = [0] * len(tree_info), []
    for nd in tree_info:
        depth[nd.id] = nd.seqlen + (depth[nd.parent] if nd.parent >= 0 else 0)
        if len(nd.requests) > 1 and depth[nd.id] > 0:
            out.append((list(nd.requests), depth[nd.id]))
    return out


def extend(q, k_buffer, v_buffer, o, kv_entries, plan, sm_scale, logit_cap=-1, o_lse=None, path="auto"):
    """Causal attention of a step's new tokens over the paged cache, which holds their prefixes and themselves (append
    first).  ``q``, ``o`` ``[tokens, q heads, head_dim]``, the pool ``[rows, kv heads, head_dim]`` (``o`` must overlap neither ``q``
    nor the pool), ``kv_entries`` the int32 table that the plan's ``kv_starts`` index (flat or ``[requests, positions]``).
    ``logit_cap`` > 0: scores become ``logit_cap * tanh(score / logit_cap)``.  ``o_lse``: optional fp32 ``[tokens, q heads]``.
    Rows of ``o`` behind the plan's tokens are left as they are.  Partial results, where the plan has them, live in memory that
    the call takes from torch's allocator on the current stream."""
    rc = _lib.call_module().extend(*_extend_call(q, k_buffer, v_buffer, o, kv_entries, plan, sm_scale, logit_cap, o_lse, path))
    if rc != 0:
        _lib.check(rc)


def _extend_call(q, k_buffer, v_buffer, o, kv_entries, plan, sm_scale, logit_cap, o_lse, path):
    if not isinstance(plan, ExtendPlan):
        raise ValueError("plan must come from fasttree_extend_preparation")
    code = _lib.EXTEND_PATHS.get(path)
    if code is None:
        raise ValueError(f"path must be one of {sorted(_lib.EXTEND_PATHS)}")
    return q, k_buffer, v_buffer, o, kv_entries, plan.table, plan._raw, sm_scale, logit_cap, o_lse, code


def path_name(q, k_buffer, v_buffer, o, kv_entries, plan, sm_scale, logit_cap=-1, o_lse=None, path="auto"):
    """Names of the kernels that :func:`extend` would launch, joined by '+'."""
    call = _extend_call(q, k_buffer, v_buffer, o, kv_entries, plan, sm_scale, logit_cap, o_lse, path)
    args = _lib.ExtendArgs.from_buffer_copy(_lib.call_module().extend_args(*call))
    name = _lib.load().ft_extend_path_name(ctypes.byref(args))
    if name is None:
        _lib.check(-1)
    return name.decode()
