"""Heads of a policy over items: scores of chosen items, a preference loss over pairs of sequences, a clipped policy loss.

The reference knows one head, the sigmoid cross entropy of a click (wd_bce_sum_fwd_bwd); these stand beside it for models whose logits
are a row of scores per position.  Each call is one entry of the C ABI (include/wd_hip.h, csrc/policy_loss.hip): loss AND gradient of
the logits, launched on the current stream of the logits' device, nothing read back, so every call can be captured into a hipGraph.
There is no autograd in between: `dlogits` goes to the backward pass of whatever made the logits, a program's own (wd_gemm_*, torch.mm).
The engine's towers are no such producer: they make their gradient from the click loss inside the step and take none from outside.

Layout of a batch: `logits` [rows, vocab] (fp32, fp16 or bf16; rows may be strided, items contiguous), `targets` int32 [rows] (outside
[0, vocab), e.g. -1: the position is no action of the policy), `seq_offs` int32 [sequences + 1], a CSR over the rows.  Results and
workspace come from torch's caching allocator on the current stream: calls on several streams share nothing.  The results of a call but for
`dlogits` are parts of one allocation with its workspace (11 floats a row, up to 2048 more where few rows are split): clone what is kept long.  Every tensor has to be
ready on the current stream; one that another stream uses later is the caller's to record there.
"""
import functools
import struct
from collections import namedtuple

import torch

from . import capi

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}     # WD_T_*
_ROWS = struct.Struct("=QqqqQQqii")                                   # wd_seq_rows_t
_PREF = struct.Struct("=QQQQQQQQqfffffiii")                           # wd_pref_t
_POLICY = struct.Struct("=QQQQQQqffffiiii")                           # wd_policy_t

PREFERENCE_KINDS = {"logistic": 0, "square": 1}                       # WD_PREF_*
POLICY_REDUCTIONS = {"sum": 0, "token_mean": 1, "sequence_mean": 2}   # WD_POLICY_*

SequenceLogp = namedtuple("SequenceLogp", "token_logp seq_logp")
PreferenceLoss = namedtuple("PreferenceLoss", "loss pair_loss difference seq_logp token_logp dlogits")
PolicyLoss = namedtuple("PolicyLoss", "loss kl clipped token_logp dlogits")


def _vector(name, t, n, dtype, device):
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.dim() != 1 or t.numel() != n or t.device != device or not t.is_contiguous():
        raise ValueError("%s: a contiguous %s tensor of %d values on %s is wanted, got %s" % (name, dtype, n, device, _what(t)))
    return t.data_ptr()


def _what(t):
    return "%s %s on %s" % (t.dtype, list(t.shape), t.device) if isinstance(t, torch.Tensor) else repr(t)


def _layout(name, t, V):
    """Row stride of a [rows, V] tensor."""
    if t.is_contiguous() and V > 0:
        return V
    step, item = t.stride()
    T = t.shape[0]
    if V < 1 or (T and V > 1 and item != 1) or (T > 1 and step < V):
        raise ValueError("%s: at least one item, items contiguous, rows not overlapping are wanted, got %s with strides %s" % (name, _what(t), t.stride()))
    return step if T > 1 else V


def _rows(logits, targets, seq_offs):
    """wd_seq_rows_t of a batch, packed, after the checks that need no device."""
    code = _DTYPES.get(logits.dtype) if isinstance(logits, torch.Tensor) and logits.dim() == 2 else None
    if code is None:
        raise ValueError("logits: a [rows, vocab] tensor of fp32, fp16 or bf16 is wanted, got %s" % _what(logits))
    T, V = logits.shape
    ld = _layout("logits", logits, V)
    dev = logits.device
    if dev.type != "cuda":
        raise capi.WdError("policy heads need a GPU (MI355X / gfx950); there is no CPU fallback: logits are on %s" % dev)
    pt = _vector("targets", targets, T, torch.int32, dev)
    N = seq_offs.numel() - 1 if isinstance(seq_offs, torch.Tensor) else 0
    po = _vector("seq_offs", seq_offs, max(N, 0) + 1, torch.int32, dev)
    return _ROWS.pack(logits.data_ptr(), ld, T, V, pt, po, N, code, 0), T, V, N, dev, code


@functools.lru_cache(maxsize=4096)
def _workspace(T, V, N, dtype):
    """Floats of workspace, by the sizes alone."""
    n = capi.call("wd_policy_workspace_floats", _ROWS.pack(16, V, T, V, 16, 16, N, dtype, 0))
    if n < 0:
        raise capi.WdError("wd_policy_workspace_floats failed (%d): %s" % (n, capi.load().wd_last_error().decode()))
    return n + (n & 1)


def _gradient(dlogits, logits):
    """(tensor or None, pointer, row stride, zero_tail) of the gradient: True: a new tensor, None / False: the loss alone."""
    if dlogits is True:
        g = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        return g, g.data_ptr(), logits.shape[1], 1       # rows of no sequence: zeros
    if dlogits is None or dlogits is False:
        return None, 0, 0, 0
    if not isinstance(dlogits, torch.Tensor) or dlogits.shape != logits.shape or dlogits.dtype is not logits.dtype or dlogits.device != logits.device:
        raise ValueError("dlogits: a tensor like logits (%s) is wanted, got %s" % (_what(logits), _what(dlogits)))
    return dlogits, dlogits.data_ptr(), _layout("dlogits", dlogits, logits.shape[1]), 0


def _call(name, dev, *args):
    """One entry of the C ABI on the current stream of `dev`."""
    if torch._C._cuda_getDevice() != dev.index:
        with torch.cuda.device(dev):
            return _call(name, dev, *args)
    capi.call(name, *args, torch._C._cuda_getCurrentRawStream(dev.index))      # the handle current_stream() wraps, without the wrapper's 1 us


def _buffer(logits, *sizes):
    """Workspace and results of a call in one allocation: its address and its parts."""
    buf = logits.new_empty(sum(sizes), dtype=torch.float32)
    return buf.data_ptr(), torch.unsafe_split_with_sizes(buf, sizes)


def sequence_logp(logits, targets, seq_offs, length_norm=False):
    """Log-probabilities of the chosen items: token_logp[r] = log softmax(logits[r])[targets[r]] (0 where the position is no action) and
    seq_logp[n], their sum over sequence n (length_norm: their mean over its actions; 0 without any)."""
    rows, T, V, N, dev, code = _rows(logits, targets, seq_offs)
    ws = _workspace(T, V, N, code)
    base, (_, token, seq) = _buffer(logits, ws, T, N)
    p = base + 4 * ws
    _call("wd_seq_logp", dev, rows, int(bool(length_norm)), p, p + 4 * T, base)
    return SequenceLogp(token, seq)


def preference_loss(logits, targets, seq_offs, ref_logp=None, weights=None, beta=0.1, kind="logistic", margin=0.0, label_smoothing=0.0,
                    length_norm=False, reduction="sum", grad_scale=1.0, dlogits=True):
    """Preference loss of pairs of sequences, 2i chosen and 2i + 1 rejected, with the gradient of the logits.

    d = (LP[2i] - ref_logp[2i]) - (LP[2i + 1] - ref_logp[2i + 1]) with LP as seq_logp of sequence_logp (which also makes ref_logp, from
    the reference model's logits); kind "logistic": -(1 - label_smoothing) log sigma(h) - label_smoothing log sigma(-h), h = beta d -
    margin; "square": (d - 1 / (2 beta))^2.  loss = sum or mean over the pairs of weights[i] times that (a pair of weight 0 adds nothing, whatever its loss).
    dlogits: True (a new tensor), a tensor like logits (rows of no sequence are left as they were; it may be `logits` itself), or None
    (the loss alone); it holds grad_scale times the gradient."""
    rows, T, V, N, dev, code = _rows(logits, targets, seq_offs)
    if kind not in PREFERENCE_KINDS or reduction not in ("sum", "mean"):
        raise ValueError("kind is one of %s, reduction sum or mean: got %r, %r" % (sorted(PREFERENCE_KINDS), kind, reduction))
    if N % 2:
        raise ValueError("preference_loss: %d sequences: pair i is sequences 2i (chosen) and 2i + 1 (rejected)" % N)
    pr = _vector("ref_logp", ref_logp, N, torch.float32, dev) if ref_logp is not None else 0
    pw = _vector("weights", weights, N // 2, torch.float32, dev) if weights is not None else 0
    g, pg, ldg, tail = _gradient(dlogits, logits)
    P = N // 2
    ws = _workspace(T, V, N, code)
    base, (_, loss, pair, diff, seq, tok) = _buffer(logits, ws, 1, P, P, N, T)
    p = base + 4 * ws
    opts = _PREF.pack(pr, pw, p, p + 4, p + 4 * (1 + P), p + 4 * (1 + 2 * P), p + 4 * (1 + 2 * P + N), pg, ldg, beta, margin, label_smoothing,
                      1.0 / max(P, 1) if reduction == "mean" else 1.0, grad_scale, PREFERENCE_KINDS[kind], int(bool(length_norm)), tail)
    _call("wd_pref_loss_fwd_bwd", dev, rows, opts, base)
    return PreferenceLoss(loss.squeeze(), pair, diff, seq, tok, g)


def policy_loss(logits, targets, seq_offs, old_logp, advantages, ref_logp=None, per_row=None, clip=(0.2, 0.2), kl_coef=0.0, reduction="token_mean",
                grad_scale=1.0, dlogits=True):
    """Clipped policy loss with a KL term to a reference policy, with the gradient of the logits.

    rho = exp(token_logp - old_logp), A = advantages by row or by sequence; each action gives -min(rho A, clip(rho, 1 - clip[0], 1 +
    clip[1]) A) + kl_coef k with k = exp(ref_logp - token_logp) - (ref_logp - token_logp) - 1.  reduction: "sum", "token_mean" (over all
    actions) or "sequence_mean" (mean over the sequences that have an action of their means).  Returns the loss, and reduced the same way
    k and the share of actions whose clipped side was taken.  old_logp and ref_logp are token_logp of sequence_logp, [rows].
    dlogits as in preference_loss.  per_row: whether advantages are [rows] or [sequences]; None: told by their number, which has to tell."""
    rows, T, V, N, dev, code = _rows(logits, targets, seq_offs)
    if reduction not in POLICY_REDUCTIONS:
        raise ValueError("reduction is one of %s: got %r" % (sorted(POLICY_REDUCTIONS), reduction))
    po = _vector("old_logp", old_logp, T, torch.float32, dev)
    if per_row is None:
        if T == N:
            raise ValueError("policy_loss: %d rows and as many sequences: say with per_row which of them the advantages belong to" % T)
        per_row = isinstance(advantages, torch.Tensor) and advantages.dim() == 1 and advantages.shape[0] == T
    pa = _vector("advantages", advantages, T if per_row else N, torch.float32, dev)
    if kl_coef and ref_logp is None:
        raise ValueError("policy_loss: a KL term needs ref_logp, the reference policy's token_logp")
    pr = _vector("ref_logp", ref_logp, T, torch.float32, dev) if ref_logp is not None else 0
    low, high = clip
    g, pg, ldg, tail = _gradient(dlogits, logits)
    ws = _workspace(T, V, N, code)
    base, (_, sums, token) = _buffer(logits, ws, 3, T)
    p = base + 4 * ws
    opts = _POLICY.pack(po, pr, pa, p, p + 12, pg, ldg, low, high, kl_coef, grad_scale, int(bool(per_row)), POLICY_REDUCTIONS[reduction], tail, 0)
    _call("wd_policy_loss_fwd_bwd", dev, rows, opts, base)
    return PolicyLoss(*sums.unbind(), token, g)
