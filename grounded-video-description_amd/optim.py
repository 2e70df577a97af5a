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

import torch

from .hip import (DTYPES, GRAD_CHUNK, GRAD_MAX_TENSORS, OPT_CHUNK, OPT_MAX_TENSORS, GradClip, GradGroup, GvdHipError, OptGroup, check,
                  lib, ptr, stream_on, stream_ptr)


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
# fp32, bf16 and fp16 gradients, mixed, clipped in place or written - unscaled - into master gradients of another type.
# ---------------------------------------------------------------------------------------------------------------------
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


def _check_grads(grads, what):
    """The gradients that have elements; dense float tensors on one GPU."""
    for i, g in enumerate(grads):
        if g.dtype not in DTYPES or g.layout != torch.strided:
            raise GvdHipError('%s: gradient %d must be a dense float32 / bfloat16 / float16 tensor, got %s %s'
                              % (what, i, g.layout, g.dtype))
        if g.device != grads[0].device:
            raise GvdHipError('%s: gradients on %s and %s' % (what, grads[0].device, g.device))
    if grads and not grads[0].is_cuda:
        raise GvdHipError('%s: the gradients are not on the GPU; there is no CPU fallback' % what)
    return [g for g in grads if g.numel()]


def _no_overlap(tensors, what):
    spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in tensors)
    for (_, end), (start, _) in zip(spans, spans[1:]):
        if start < end:
            raise GvdHipError('%s: two of the tensors to be written share memory' % what)


def _grad_groups(grads, out):
    """Launch arguments of at most GRAD_MAX_TENSORS tensors each; out: the tensors to be written (None: the norm alone)."""
    groups = []
    for k in range(0, len(grads), GRAD_MAX_TENSORS):
        part = grads[k:k + GRAD_MAX_TENSORS]
        g = GradGroup()
        g.count = len(part)
        ns = [t.numel() for t in part]
        g.src[:len(part)] = [t.data_ptr() for t in part]
        g.n[:len(part)] = ns
        g.src_type[:len(part)] = [DTYPES[t.dtype] for t in part]
        at, firsts = 0, [0]
        for n in ns:
            at += -(-n // GRAD_CHUNK)
            firsts.append(at)
        g.chunk0[:len(part) + 1] = firsts
        if out is not None:
            w = out[k:k + GRAD_MAX_TENSORS]
            g.dst[:len(part)] = [t.data_ptr() for t in w]
            g.dst_type[:len(part)] = [DTYPES[t.dtype] for t in w]
        groups.append(g)
    return groups


def _norm_and_scale(grads, out, max_norm, inv_scale, error_if_nonfinite, what):
    """grads: live, dense.  The norm (device scalar); out (tensors like grads) = the clipped gradients, None = the norm alone."""
    dev = grads[0].device
    norm = torch.empty((), dtype=torch.float32, device=dev)
    groups = _grad_groups(grads, out)
    l = lib()
    parts = []
    for g in groups:
        n = l.gvd_grad_parts(C.byref(g))
        if n <= 0:
            raise GvdHipError('%s: the gradients are too large for one call' % what)
        parts.append(n)
    partials = torch.empty(sum(parts), dtype=torch.float64, device=dev)
    c = GradClip(max_norm, inv_scale)
    with torch.cuda.device(dev):
        st = stream_on(dev)
        at = partials.data_ptr()
        for g, n in zip(groups, parts):
            check(l.gvd_grad_sumsq(C.byref(g), at, st), 'gvd_grad_sumsq')
            at += 8 * n
        if out is None or error_if_nonfinite:
            check(l.gvd_grad_scale(C.byref(GradGroup()), C.byref(c), ptr(partials), sum(parts), ptr(norm), st), 'gvd_grad_scale')
            if error_if_nonfinite and not bool(torch.isfinite(norm)):
                raise RuntimeError('%s: the total norm of the gradients is not finite (%s); they were not clipped' % (what, float(norm)))
        if out is not None:
            for i, g in enumerate(groups):
                check(l.gvd_grad_scale(C.byref(g), C.byref(c), ptr(partials), sum(parts), None if i else ptr(norm), st),
                      'gvd_grad_scale')
    return norm


def _check_clip(max_norm, inv_scale, what):
    max_norm, inv_scale = float(max_norm), float(inv_scale)
    if not max_norm >= 0.0:
        raise GvdHipError('%s: max_norm must be >= 0, got %r' % (what, max_norm))
    if not 0.0 < inv_scale < math.inf:
        raise GvdHipError('%s: inv_scale must be positive and finite, got %r' % (what, inv_scale))
    return max_norm, inv_scale


@torch.no_grad()
def grad_norm(grads, inv_scale=1.0):
    """inv_scale * the L2 norm of all elements of all tensors, a float32 scalar on their device (0 for none).  Summed in fp64 in a
    fixed order.  fp32 / bf16 / fp16 tensors of any strides, on one GPU."""
    what = 'grad_norm'
    _, inv_scale = _check_clip(0.0, inv_scale, what)
    grads = list(grads)
    live = _check_grads(grads, what)
    if not live:
        return torch.zeros((), device=grads[0].device if grads else 'cuda')
    return _norm_and_scale([g if _dense(g) else g.contiguous() for g in live], None, 0.0, inv_scale, False, what)


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
    if out is not None:
        out = list(out)
        if len(out) != len(grads):
            raise GvdHipError('%s: %d gradients, %d results' % (what, len(grads), len(out)))
        for i, (g, o) in enumerate(zip(grads, out)):
            if o.device != g.device or o.dtype not in DTYPES or o.shape != g.shape:
                raise GvdHipError('%s: result %d must be a float32 / bfloat16 / float16 tensor %s on %s' % (what, i, tuple(g.shape),
                                                                                                            g.device))
        out = [o for o in out if o.numel()]
    live = _check_grads(grads, what)
    if not live:
        return torch.zeros((), device=grads[0].device if grads else 'cuda')
    if out is None:
        src = [g if _dense(g) else g.contiguous() for g in live]
        dst, back = src, [(g, s) for g, s in zip(live, src) if s is not g]
        for g, _ in back:
            if any(s == 0 and n > 1 for s, n in zip(g.stride(), g.shape)):
                raise GvdHipError('%s: a gradient of strides %s cannot be clipped in place' % (what, g.stride()))
    else:
        # element i of a result belongs to element i of its gradient: same order in memory, or both in row-major order
        src, dst, back = [], [], []
        for g, o in zip(live, out):
            if any(s == 0 and n > 1 for s, n in zip(o.stride(), o.shape)):
                raise GvdHipError('%s: a result of strides %s cannot be written' % (what, o.stride()))
            same = g.stride() == o.stride() and _dense(g)
            src.append(g if same else g.contiguous())
            dst.append(o if same or o.is_contiguous() else torch.empty_like(o, memory_format=torch.contiguous_format))
            if dst[-1] is not o:
                back.append((o, dst[-1]))
    _no_overlap(dst, what)
    if out is not None:
        _no_partial_alias(src, dst, what)
    norm = _norm_and_scale(src, dst, max_norm, inv_scale, error_if_nonfinite, what)
    for o, d in back:
        o.copy_(d)
    written = live if out is None else out
    torch.autograd.graph.increment_version([t for t in written if not t.is_inference()])
    return norm


def _no_partial_alias(src, dst, what):
    """A result is its own gradient (clipped in place) or shares no memory with any gradient."""
    spans = sorted([(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), i, 0) for i, t in enumerate(src)] +
                   [(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), i, 1) for i, t in enumerate(dst)])
    open_ = []
    for a, b, i, written in spans:
        open_ = [s for s in open_ if s[1] > a]
        for a2, b2, j, w2 in open_:
            own = i == j and (a, b) == (a2, b2) and src[i].dtype == dst[i].dtype
            if written != w2 and not own:
                raise GvdHipError('%s: a result shares memory with a gradient that is not its own' % what)
        open_.append((a, b, i, written))


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """torch.nn.utils.clip_grad_norm_ (main.py:265) on the library's kernels: the gradients of `parameters` (a tensor or an
    iterable of tensors; those without a gradient are passed over) are scaled in place by min(1, max_norm / (norm + 1e-6)).
    Returns the norm before clipping.  The L2 norm only."""
    if float(norm_type) != 2.0:
        raise GvdHipError('clip_grad_norm_: the L2 norm only (norm_type = 2), got %r' % (norm_type,))
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    return clip_grads([p.grad for p in parameters if p.grad is not None], max_norm, error_if_nonfinite=error_if_nonfinite)
