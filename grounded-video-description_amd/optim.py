"""The optimiser step of main.train (main.py:263-266: `clip_grad_norm_(model.parameters(), opt.grad_clip)` followed by
`optimizer.step()` of torch.optim.Adam) on the library's own multi-tensor kernels (csrc/optim.hip).

`ClipAdam` IS a torch.optim.Adam (same constructor, param groups, `state` entries 'step' / 'exp_avg' / 'exp_avg_sq',
`state_dict()` / `load_state_dict()` interchangeable with the reference's optimizer); only `step()` is replaced, and
`step_clipped(max_norm)` fuses the gradient clipping into it: the total norm comes from ordered per-chunk partial sums,
the clip factor stays on the device, and every gradient is scaled while the Adam pass reads it - the clipped gradients are
never written back (so, unlike after clip_grad_norm_, `.grad` still holds the UNCLIPPED gradients afterwards).
"""
import ctypes as C
import math
import operator

import numpy as np
import torch

from . import hip
from .hip import (DTYPES, GRAD_CHUNK, GRAD_MAX_TENSORS, OPT_CHUNK, OPT_MAX_TENSORS, GradClip, GradGroup, GvdHipError, OptGroup, check,
                  lib, ptr, run_on, stream_ptr)


class ClipAdam(torch.optim.Adam):
    def __init__(self, params, **kw):
        for k in ('amsgrad', 'maximize', 'capturable', 'differentiable', 'decoupled_weight_decay'):
            if kw.get(k):
                raise ValueError('ClipAdam: %s is not supported' % k)
        kw.pop('fused', None)
        kw.pop('foreach', None)
        super().__init__(params, foreach=False, fused=False, **kw)
        self._partials = None
        self._clip = None
        self._stepped = []          # state dicts whose step counter the last step_clipped() advanced (rollback)

    # ------------------------------------------------------------------------------------------------------------
    def _live(self):
        """[(param, grad, group)] of the parameters that take part in this step (those with a gradient), in group order."""
        out = []
        for group in self.param_groups:
            for p in group['params']:
                if p.grad is None:
                    continue
                if p.grad.is_sparse or p.dtype != torch.float32 or not p.is_cuda:
                    raise GvdHipError('ClipAdam: dense fp32 GPU parameters only (there is no CPU path)')
                if not p.is_contiguous():
                    raise GvdHipError('ClipAdam: parameters must be contiguous')
                if not p.grad.is_contiguous():       # (autograd lays gradients out like their parameter; be safe)
                    p.grad = p.grad.contiguous()
                out.append((p, p.grad, group))
        return out

    @staticmethod
    def _launches(items):
        """Split [(tensors..., n)] into launches of at most OPT_MAX_TENSORS tensors; yields (first_chunk, OptGroup, idx)."""
        first = 0
        for i0 in range(0, len(items), OPT_MAX_TENSORS):
            part = items[i0:i0 + OPT_MAX_TENSORS]
            g = OptGroup()
            g.count = len(part)
            g.part0 = first
            c = 0
            for t, it in enumerate(part):
                g.chunk0[t] = c
                c += -(-it['n'] // OPT_CHUNK)
                g.n[t] = it['n']
                g.g[t] = it['g'].data_ptr()
                ok = it['g'].data_ptr() % 16 == 0
                for key in ('p', 'm', 'v'):
                    if key in it:
                        getattr(g, key)[t] = it[key].data_ptr()
                        ok = ok and it[key].data_ptr() % 16 == 0
                g.vec_ok[t] = 1 if ok else 0
                g.lr[t] = it.get('lr', 0.0)
                g.bc1[t] = it.get('bc1', 1.0)
                g.bc2_sqrt[t] = it.get('bc2_sqrt', 1.0)
            g.chunk0[len(part)] = c
            yield g
            first += c

    def grad_norm_and_clip(self, live, max_norm):
        """Device tensor [2] = (total L2 norm of the live gradients, min(1, max_norm / (norm + 1e-6)))."""
        items = [{'g': g, 'n': g.numel()} for _, g, _ in live]
        total = sum(-(-it['n'] // OPT_CHUNK) for it in items)
        dev = live[0][0].device
        if self._partials is None or self._partials.numel() < total or self._partials.device != dev:
            self._partials = torch.empty(total, dtype=torch.float32, device=dev)
        self._clip = torch.empty(2, dtype=torch.float32, device=dev)     # (fresh: a caller may keep last step's norm)
        for g in self._launches(items):
            check(lib().gvd_sumsq_partials(C.byref(g), ptr(self._partials), stream_ptr()), 'gvd_sumsq_partials')
        check(lib().gvd_clip_coef(ptr(self._partials), total, float(max_norm), ptr(self._clip), stream_ptr()),
              'gvd_clip_coef')
        return self._clip

    @torch.no_grad()
    def step_clipped(self, max_norm=None, closure=None, skip=None):
        """clip_grad_norm_(all parameters of all groups, max_norm) + Adam.step() in one go.  Returns the pre-clip total
        gradient norm as a device scalar (None without clipping).
        skip: optional device int32 vector; if any element is non-zero WHEN THE KERNELS RUN, the update kernels change
        nothing (the norm is still computed).  The caller reads the vector afterwards and, if it was raised, calls
        rollback_step_counts() - so the optimiser can be enqueued before the flags that validate the step are known."""
        if closure is not None:
            raise ValueError('ClipAdam: closures are not supported')
        live = self._live()
        self._stepped = []
        if not live:
            return None
        if skip is not None:
            assert skip.is_cuda and skip.dtype == torch.int32 and skip.is_contiguous() and 0 < skip.numel() <= 64
        clip = self.grad_norm_and_clip(live, max_norm) if max_norm is not None else None
        # one launch list per (betas, eps, weight_decay) combination (the recipe has one: main.py:660-677)
        by_hyper = {}
        for p, g, group in live:
            st = self.state[p]
            if len(st) == 0:
                st['step'] = torch.tensor(0.0, dtype=torch.float32)
                st['exp_avg'] = torch.zeros_like(p, memory_format=torch.preserve_format)
                st['exp_avg_sq'] = torch.zeros_like(p, memory_format=torch.preserve_format)
            if st['step'].is_cuda:       # (a state_dict written by torch's fused Adam keeps `step` on the device)
                st['step'] = st['step'].detach().cpu()
            st['step'] += 1
            self._stepped.append(st)
            t = float(st['step'])
            b1, b2 = group['betas']
            key = (b1, b2, group['eps'], group['weight_decay'])
            by_hyper.setdefault(key, []).append({
                'p': p, 'g': g, 'm': st['exp_avg'], 'v': st['exp_avg_sq'], 'n': p.numel(), 'lr': float(group['lr']),
                'bc1': 1.0 - b1 ** t, 'bc2_sqrt': math.sqrt(1.0 - b2 ** t)})
        for (b1, b2, eps, wd), items in by_hyper.items():
            for g in self._launches(items):
                check(lib().gvd_adam_step(C.byref(g), ptr(clip), ptr(skip), 0 if skip is None else skip.numel(), b1, b2, eps,
                                          wd, stream_ptr()), 'gvd_adam_step')
        # the kernels wrote p / exp_avg / exp_avg_sq through raw pointers: tell autograd's version counters, as torch's
        # in-place Adam does - anything keyed on `_version` (att_model._packed: the re-laid-out inference weights; saved
        # tensors of a retained graph) must see that the parameters changed
        torch.autograd.graph.increment_version([t for p, _, _ in live
                                                for t in (p, self.state[p]['exp_avg'], self.state[p]['exp_avg_sq'])])
        return None if clip is None else clip[0]

    def rollback_step_counts(self):
        """Undo the step-counter advance of the last step_clipped() (whose device side was skipped: `skip` was raised)."""
        for st in self._stepped:
            st['step'] -= 1
        self._stepped = []

    def step(self, closure=None):
        self.step_clipped(None, closure)


# ---------------------------------------------------------------------------------------------------------------------
# The global gradient norm and clipping as operators of their own (csrc/grad_clip.hip), for optimisers other than ClipAdam:
# fp32, bf16 and fp16 gradients, mixed, clipped in place or written - unscaled - into master gradients of another type.  What
# is looked at per tensor goes through map() and numpy: with hundreds of small gradients the host is what a call waits for.
# ---------------------------------------------------------------------------------------------------------------------
_DTYPE, _SHAPE = operator.attrgetter('dtype'), operator.attrgetter('shape')
_T = torch.Tensor
_GROUP_FIELDS = {f: (getattr(GradGroup, f).offset, t) for f, t in (('src', np.int64), ('dst', np.int64), ('n', np.int64),
                                                                   ('chunk0', np.uint32), ('src_type', np.uint8), ('dst_type', np.uint8))}


def _dense(t):
    """t's elements fill one stretch of memory, each at a place of its own (in whatever order)."""
    if t.is_contiguous():
        return True
    step = 1
    for s, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if s != step:
            return False
        step *= n
    return True


def _repeats(t):
    """Several elements of t share a place."""
    return any(s == 0 and n > 1 for s, n in zip(t.stride(), t.shape))


class _Tensors:
    """Addresses, sizes and type codes of a list of dense float tensors on one GPU."""

    def __init__(self, tensors, what, like=None):
        types = list(map(_DTYPE, tensors))
        if types.count(types[0]) == len(types) and types[0] in DTYPES:
            self.code = np.full(len(types), DTYPES[types[0]], np.uint8)
        else:
            self.code = np.array([DTYPES.get(t, 255) for t in types], np.uint8)
            if (self.code == 255).any():
                i = int((self.code == 255).argmax())
                raise GvdHipError('%s: tensor %d must be float32 / bfloat16 / float16, got %s' % (what, i, types[i]))
        devices = set(map(_T.get_device, tensors))
        if len(devices) > 1:
            raise GvdHipError('%s: tensors on several devices (%s)' % (what, sorted(devices)))
        if not tensors[0].is_cuda:
            raise GvdHipError('%s: the tensors are not on the GPU; there is no CPU fallback' % what)
        self.n = like.n if like is not None else np.array(list(map(_T.numel, tensors)), np.int64)
        self.ptr = np.array(list(map(_T.data_ptr, tensors)), np.int64)
        self.end = self.ptr + self.n * np.where(self.code == 0, 4, 2)


def _strided(tensors, what):
    for i, t in enumerate(tensors):
        if t.layout != torch.strided:
            raise GvdHipError('%s: tensor %d must be dense, got %s' % (what, i, t.layout))


def _all_contiguous(tensors, what):
    try:
        return all(map(_T.is_contiguous, tensors))
    except RuntimeError:                                 # (a sparse tensor)
        _strided(tensors, what)
        raise


def _any_overlap(starts, ends):
    order = np.argsort(starts)
    return len(order) > 1 and bool((np.maximum.accumulate(ends[order])[:-1] > starts[order][1:]).any())


def _check_written(src, dst, what):
    """No two written tensors share memory; a result is its own gradient or shares memory with none."""
    if src is dst:
        if _any_overlap(dst.ptr, dst.end):
            raise GvdHipError('%s: two of the tensors to be written share memory' % what)
        return
    other = ~((src.ptr == dst.ptr) & (src.code == dst.code))
    if not _any_overlap(np.concatenate([dst.ptr, src.ptr[other]]), np.concatenate([dst.end, src.end[other]])):
        return
    if _any_overlap(dst.ptr, dst.end):
        raise GvdHipError('%s: two of the tensors to be written share memory' % what)
    # (gradients may overlap each other, results nothing: look at each gradient's neighbours among the results)
    order = np.argsort(dst.ptr)
    starts, ends = dst.ptr[order], dst.end[order]
    k = np.searchsorted(ends, src.ptr[other], side='right')          # the first result that ends behind the gradient's start
    hit = (k < len(starts)) & (starts[np.minimum(k, len(starts) - 1)] < src.end[other])
    if bool(hit.any()):
        raise GvdHipError('%s: a result shares memory with a gradient that is not its own' % what)


def _grad_groups(src, dst):
    """Launch arguments of at most GRAD_MAX_TENSORS tensors each; dst None: the norm alone."""
    groups = []
    chunks = -(-src.n // GRAD_CHUNK)
    for k in range(0, len(src.n), GRAD_MAX_TENSORS):
        part = slice(k, k + GRAD_MAX_TENSORS)
        g = GradGroup()
        count = g.count = len(src.n[part])

        def put(field, values, at=0):
            offset, dtype = _GROUP_FIELDS[field]
            np.frombuffer(g, dtype, count + at, offset)[at:] = values
        put('src', src.ptr[part])
        put('n', src.n[part])
        put('src_type', src.code[part])
        put('chunk0', np.cumsum(chunks[part]), 1)
        if dst is not None:
            put('dst', dst.ptr[part])
            put('dst_type', dst.code[part])
        groups.append(g)
    return groups


def _norm_and_scale(dev, src, dst, max_norm, inv_scale, error_if_nonfinite, what):
    """The norm of src (device scalar); dst = the clipped gradients, None = the norm alone."""
    if int(src.n.max()) > GRAD_CHUNK * 0x7fffffff // len(src.n):
        raise GvdHipError('%s: the gradients are too large for one call' % what)
    norm = torch.empty((), dtype=torch.float32, device=dev)
    groups = _grad_groups(src, dst)
    l = lib()
    parts = [l.gvd_grad_parts(C.byref(g)) for g in groups]
    if min(parts) <= 0:
        raise GvdHipError('%s: gvd_grad_parts refused the gradients' % what)
    total = sum(parts)
    partials = torch.empty(total, dtype=torch.float64, device=dev)
    c = GradClip(max_norm, inv_scale)
    at = first = partials.data_ptr()
    for g, n in zip(groups, parts):
        run_on(dev, l.gvd_grad_sumsq, 'gvd_grad_sumsq', C.byref(g), at)
        at += 8 * n
    if dst is None or error_if_nonfinite:
        run_on(dev, l.gvd_grad_scale, 'gvd_grad_scale', C.byref(GradGroup()), C.byref(c), first, total, norm.data_ptr())
        if error_if_nonfinite and not bool(torch.isfinite(norm)):
            raise RuntimeError('%s: the total norm of the gradients is not finite (%s); they were not clipped' % (what, float(norm)))
    if dst is not None:
        for i, g in enumerate(reversed(groups)):       # (backwards: what was read last is still in the cache)
            run_on(dev, l.gvd_grad_scale, 'gvd_grad_scale', C.byref(g), C.byref(c), first, total, None if i else norm.data_ptr())
    return norm


def _check_clip(max_norm, inv_scale, what):
    max_norm, inv_scale = float(max_norm), float(inv_scale)
    if not max_norm >= 0.0:
        raise GvdHipError('%s: max_norm must be >= 0, got %r' % (what, max_norm))
    if not 0.0 < inv_scale < math.inf:
        raise GvdHipError('%s: inv_scale must be positive and finite, got %r' % (what, inv_scale))
    return max_norm, inv_scale


def _no_gradients():
    return torch.zeros((), device='cuda')


@torch.no_grad()
def grad_norm(grads, inv_scale=1.0):
    """inv_scale * the L2 norm of all elements of all tensors, a float32 scalar on their device (0 for none).  Summed in fp64 in a
    fixed order.  fp32 / bf16 / fp16 tensors of any strides, on one GPU."""
    what = 'grad_norm'
    _, inv_scale = _check_clip(0.0, inv_scale, what)
    grads = list(grads)
    if not _all_contiguous(grads, what):
        _strided(grads, what)
        grads = [g if _dense(g) else g.contiguous() for g in grads]
    if not grads:
        return _no_gradients()
    t, device = _Tensors(grads, what), grads[0].device
    if not t.n.all():
        grads = [g for g in grads if g.numel()]
        if not grads:
            return torch.zeros((), device=device)
        t = _Tensors(grads, what)
    return _norm_and_scale(device, t, None, 0.0, inv_scale, False, what)


@torch.no_grad()
def clip_grads(grads, max_norm, out=None, inv_scale=1.0, error_if_nonfinite=False):
    """grads * min(1, max_norm / (norm + 1e-6)) * inv_scale, where norm = inv_scale * the L2 norm of them all.

    In place, or into `out` (one tensor per gradient, of its shape, any of the three types: 16-bit gradients of a scaled loss go
    unscaled and clipped into fp32 master gradients; views of a flat buffer are fine).  Returns the norm before clipping, a
    float32 scalar on the device; nothing waits for the GPU unless error_if_nonfinite is set, which raises RuntimeError before
    anything is written if the norm is NaN or infinite.  Otherwise a NaN norm makes every gradient NaN and an infinite one every
    finite gradient 0, as torch.nn.utils.clip_grad_norm_ does.  One GPU; tensors to be written must not share memory."""
    what = 'clip_grads'
    max_norm, inv_scale = _check_clip(max_norm, inv_scale, what)
    grads = list(grads)
    written = grads if out is None else list(out)
    if out is not None:
        if len(written) != len(grads):
            raise GvdHipError('%s: %d gradients, %d results' % (what, len(grads), len(written)))
        if list(map(_SHAPE, grads)) != list(map(_SHAPE, written)):
            i = [g.shape == o.shape for g, o in zip(grads, written)].index(False)
            raise GvdHipError('%s: result %d must be of shape %s, got %s' % (what, i, tuple(grads[i].shape), tuple(written[i].shape)))
    plain = _all_contiguous(grads, what) and (out is None or _all_contiguous(written, what))
    if not plain:
        _strided(grads, what)
        _strided(written, what)
    if not grads:
        return _no_gradients()
    s = _Tensors(grads, what)
    d = s if out is None else _Tensors(written, what, s)
    if out is not None and grads[0].device != written[0].device:
        raise GvdHipError('%s: gradients on %s, results on %s' % (what, grads[0].device, written[0].device))
    device = grads[0].device
    if not s.n.all():
        keep = s.n.nonzero()[0].tolist()
        if not keep:
            return torch.zeros((), device=device)
        return clip_grads([grads[i] for i in keep], max_norm, None if out is None else [written[i] for i in keep], inv_scale,
                          error_if_nonfinite)
    back = []
    if not plain:
        # element i of a result belongs to element i of its gradient: same order in memory, or both in row-major order
        src, dst = [], []
        for g, o in zip(grads, written):
            if _repeats(o):
                raise GvdHipError('%s: a tensor of strides %s cannot be written' % (what, o.stride()))
            same = g.stride() == o.stride() and _dense(g)
            src.append(g if same else g.contiguous())
            dst.append(o if same or o.is_contiguous() else src[-1] if o is g else torch.empty_like(o, memory_format=torch.contiguous_format))
            if dst[-1] is not o:
                back.append((o, dst[-1]))
        s = _Tensors(src, what)
        d = s if all(map(operator.is_, src, dst)) else _Tensors(dst, what, s)
        for o, _ in back:
            _check_scattered(o, grads + written, what)
    _check_written(s, d, what)
    norm = _norm_and_scale(device, s, d, max_norm, inv_scale, error_if_nonfinite, what)
    for o, x in back:
        o.copy_(x)
    hip.written(written)
    return norm


def _check_scattered(o, tensors, what):
    """`o`, a result with gaps that is written by way of a copy, lies apart from every other tensor of the call."""
    span = lambda t: (t.data_ptr(), t.data_ptr() + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size())  # noqa: E731
    first, last = span(o)
    for t in tensors:
        a, b = span(t)
        if t is not o and a < last and first < b:
            raise GvdHipError('%s: a result of strides %s lies among other tensors of the call' % (what, o.stride()))


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """torch.nn.utils.clip_grad_norm_ (main.py:265) on the library's kernels: the gradients of `parameters` (a tensor or an
    iterable of tensors; those without a gradient are passed over) are scaled in place by min(1, max_norm / (norm + 1e-6)).
    Returns the norm before clipping.  The L2 norm only."""
    if float(norm_type) != 2.0:
        raise GvdHipError('clip_grad_norm_: the L2 norm only (norm_type = 2), got %r' % (norm_type,))
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    return clip_grads([p.grad for p in parameters if p.grad is not None], max_norm, error_if_nonfinite=error_if_nonfinite)
