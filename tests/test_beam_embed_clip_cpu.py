"""CPU: the token-side operators (embedding lookup, gradient clipping, beam selection, state reordering) refuse what they do not
take - the Python entry points before they touch a GPU, the C entries before they launch anything - and the structs of their
C-ABI have the header's layout."""
import ctypes as C
import os
import subprocess

import pytest
import torch

from gvd_amd import hip, ops, optim

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _refused(text, fn, *a, **k):
    with pytest.raises(hip.GvdHipError, match=text):
        fn(*a, **k)


def test_struct_layouts_match_the_header(tmp_path):
    pairs = {'gvd_grad_group': hip.GradGroup, 'gvd_grad_clip': hip.GradClip, 'gvd_beam_select_args': hip.BeamSelectArgs,
             'gvd_reorder_tensor': hip.ReorderTensor, 'gvd_reorder_group': hip.ReorderGroup}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "gvd_hip.h"', 'int main(void) {']
    for cname, cls in pairs.items():
        lines.append('  printf("%s size %%zu\\n", sizeof(%s));' % (cname, cname))
        for fname, _ in cls._fields_:
            lines.append('  printf("%s %s %%zu\\n", offsetof(%s, %s));' % (cname, fname, cname, fname))
    for name in ('GVD_GRAD_MAX_TENSORS', 'GVD_GRAD_CHUNK', 'GVD_BEAM_SELECT_MAX', 'GVD_REORDER_MAX_TENSORS', 'GVD_EMBEDDING_MAX'):
        lines.append('  printf("const %s %%d\\n", %s);' % (name, name))
    src = tmp_path / 'layout.c'
    src.write_text('\n'.join(lines + ['  return 0;', '}']))
    exe = tmp_path / 'layout'
    subprocess.check_call(['gcc', '-I', os.path.join(ROOT, 'include'), str(src), '-o', str(exe)])
    got = {tuple(ln.split()[:2]): int(ln.split()[2]) for ln in subprocess.check_output([str(exe)]).decode().split('\n') if ln.strip()}
    for cname, cls in pairs.items():
        assert got[(cname, 'size')] == C.sizeof(cls), cname
        for fname, _ in cls._fields_:
            assert got[(cname, fname)] == getattr(cls, fname).offset, (cname, fname)
    assert got[('const', 'GVD_GRAD_MAX_TENSORS')] == hip.GRAD_MAX_TENSORS
    assert got[('const', 'GVD_GRAD_CHUNK')] == hip.GRAD_CHUNK == hip.lib().gvd_grad_chunk()
    assert got[('const', 'GVD_BEAM_SELECT_MAX')] == hip.BEAM_SELECT_MAX
    assert got[('const', 'GVD_REORDER_MAX_TENSORS')] == hip.REORDER_MAX_TENSORS
    assert got[('const', 'GVD_EMBEDDING_MAX')] == hip.EMBEDDING_MAX
    # a launch's arguments stay inside 4 KiB
    assert C.sizeof(hip.GradGroup) + C.sizeof(hip.GradClip) + 32 <= 4096 and C.sizeof(hip.ReorderGroup) + 32 <= 4096


def test_embedding_refusals():
    w, t = torch.zeros(7, 4), torch.zeros(3, dtype=torch.int64)
    _refused('int64 or int32', ops.embedding, t.float(), w)
    _refused('int64 or int32', ops.embedding, t.to(torch.uint8), w)
    _refused('2-D float32', ops.embedding, t, w.double())
    _refused('2-D float32', ops.embedding, t, w.view(7, 2, 2))
    _refused('act must be', ops.embedding, t, w, act=2)
    _refused('padding_idx 7', ops.embedding, t, w, padding_idx=7)
    _refused('padding_idx -8', ops.embedding, t, w, padding_idx=-8)
    _refused('no rows', ops.embedding, t, torch.zeros(0, 4))
    _refused('at most', ops.embedding, t, torch.zeros(1, 1).expand(1 << 26, 1))
    _refused('at most', ops.embedding, t, torch.zeros(1, 1).expand(1, (1 << 20) + 1))
    _refused('no CPU fallback', ops.embedding, t, w)
    _refused('no CPU fallback', ops.embedding, t.int(), w.bfloat16(), padding_idx=-7)


def test_clip_refusals():
    g = [torch.zeros(5), torch.zeros(2, 3)]
    _refused('max_norm', optim.clip_grads, g, -1.0)
    _refused('max_norm', optim.clip_grads, g, float('nan'))
    for inv in (0.0, -1.0, float('inf'), float('nan')):
        _refused('inv_scale', optim.clip_grads, g, 1.0, inv_scale=inv)
        _refused('inv_scale', optim.grad_norm, g, inv_scale=inv)
    _refused('2 gradients, 1 results', optim.clip_grads, g, 1.0, out=g[:1])
    _refused('result 1', optim.clip_grads, g, 1.0, out=[torch.zeros(5), torch.zeros(3, 2)])
    _refused('no CPU fallback', optim.clip_grads, g, 1.0, out=[torch.zeros(5).double(), torch.zeros(2, 3)])
    _refused('tensor 1 must be', optim.clip_grads, [g[0], g[1].double()], 1.0)
    _refused('tensor 0 must be', optim.grad_norm, [torch.zeros(4, 4).to_sparse()])
    _refused('no CPU fallback', optim.clip_grads, g, 1.0)
    _refused('no CPU fallback', optim.grad_norm, g)
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.ones(3)
    _refused('L2 norm only', optim.clip_grad_norm_, [p], 1.0, norm_type=float('inf'))
    _refused('no CPU fallback', optim.clip_grad_norm_, p, 1.0)


def test_beam_select_refusals():
    x, s = torch.zeros(6, 50), torch.zeros(2, 3)
    _refused('float16 and scores', ops.beam_select, x.double(), s)
    _refused('float16 and scores', ops.beam_select, x, s.half())
    _refused('float16 and scores', ops.beam_select, x, s.view(-1))
    _refused('do not fit', ops.beam_select, torch.zeros(5, 50), s)
    _refused('do not fit', ops.beam_select, torch.zeros(3, 2, 50), s)
    _refused('needs 1 <= beams', ops.beam_select, x, s, width=0)
    _refused('needs 1 <= beams', ops.beam_select, x, s, width=33)
    _refused('needs 1 <= beams', ops.beam_select, torch.zeros(6, 1), s, width=4)
    _refused('needs 1 <= beams', ops.beam_select, torch.zeros(33, 50), torch.zeros(1, 33))
    _refused('needs 1 <= beams', ops.beam_select, torch.zeros(0, 50), torch.zeros(0, 3))
    _refused('needs 1 <= beams', ops.beam_select, torch.zeros(1, 1).expand(65536, 1), torch.zeros(32768, 2))
    _refused('finished must be', ops.beam_select, x, s, finished=torch.zeros(2, 3), eos=0)
    _refused('finished must be', ops.beam_select, x, s, finished=torch.zeros(3, 2, dtype=torch.uint8), eos=0)
    _refused('eos must be', ops.beam_select, x, s, finished=torch.zeros(2, 3, dtype=torch.uint8))
    for eos in (-1, 50):
        _refused('eos must be', ops.beam_select, x, s, eos=eos)
    _refused('no CPU fallback', ops.beam_select, x, s, eos=0)


def test_reorder_refusals():
    x, p = torch.zeros(2, 6, 4), torch.zeros(6, dtype=torch.int64)
    _refused('parent must be int64', ops.reorder_rows, [x], p.int(), dim=1)
    _refused('no dimension 3', ops.reorder_rows, [x], p, dim=3)
    _refused('state 1 has 5 rows', ops.reorder_rows, [x, torch.zeros(2, 5)], p, dim=1)
    _refused('1 states, 0 results', ops.reorder_rows, [x], p, dim=1, out=[])
    _refused('result 0 must be', ops.reorder_rows, [x], p, dim=1, out=[torch.zeros(2, 5, 4)])
    _refused('result 0 must be', ops.reorder_rows, [x], p, dim=1, out=[x.double()])
    _refused('whole rows', ops.reorder_rows, [x], p, dim=1, out=[torch.zeros(2, 1, 4).expand(2, 6, 4)])
    _refused('whole rows', ops.reorder_rows, [x], p, dim=1, out=[torch.zeros(2, 4, 6).transpose(1, 2)])
    _refused('no rows', ops.reorder_rows, [torch.zeros(0, 4)], p)
    _refused('no CPU fallback', ops.reorder_rows, [x], p, dim=1)


def test_c_entries_refuse_before_they_launch():
    """-1 (unsupported) for bad sizes and addresses; the addresses here are never read."""
    l, a = hip.lib(), C.c_void_p(4096)
    assert l.gvd_embedding_fwd(a, 1, 4, a, 8, 10, 8, 3, 1.0, 0, a, 8, None) == -1            # type
    assert l.gvd_embedding_fwd(a, 1, 4, a, 7, 10, 8, 0, 1.0, 0, a, 8, None) == -1            # row stride
    assert l.gvd_embedding_fwd(a, 1, 0, a, 8, 10, 8, 0, 1.0, 0, a, 8, None) == -1
    assert l.gvd_embedding_fwd(None, 1, 4, a, 8, 10, 8, 0, 1.0, 0, a, 8, None) == -1
    assert l.gvd_embedding_fwd(a, 1, (1 << 25) + 1, a, 8, 10, 8, 0, 1.0, 0, a, 8, None) == -1
    need = l.gvd_embedding_bwd_workspace_bytes(5000, 50, 8)
    assert need > 0 and l.gvd_embedding_bwd_workspace_bytes(1000, 50, 8) == 0 and l.gvd_embedding_bwd_workspace_bytes(0, 50, 8) == 0
    assert l.gvd_embedding_bwd(a, 1, 5000, a, 8, a, 8, 50, 8, 0, 1.0, 0, -1, a, a, need - 1, None) == -1
    assert l.gvd_embedding_bwd(a, 1, 5000, a, 8, None, 8, 50, 8, 0, 1.0, 1, -1, a, a, need, None) == -1    # act without its table
    assert l.gvd_embedding_bwd(a, 1, 5000, a, -8, a, 8, 50, 8, 0, 1.0, 0, -1, a, a, need, None) == -1
    assert l.gvd_embedding_bwd(a, 1, 5000, a, 8, a, 8, 50, 8, 0, 1.0, 0, -1, a, C.c_void_p(4100), need, None) == -1

    g = hip.GradGroup()
    c = hip.GradClip(1.0, 1.0)
    assert l.gvd_grad_sumsq(C.byref(g), a, None) == -1                                       # nothing in it
    g.count, g.n[0], g.src[0], g.dst[0], g.chunk0[1] = 1, 9000, 4096, 4096, 2
    assert l.gvd_grad_parts(C.byref(g)) == 2
    g.chunk0[1] = 1
    assert l.gvd_grad_parts(C.byref(g)) == -1 and l.gvd_grad_sumsq(C.byref(g), a, None) == -1
    g.chunk0[1] = 2
    g.src[0] = 4098                                                                          # not on an element
    assert l.gvd_grad_sumsq(C.byref(g), a, None) == -1
    g.src[0] = 4096
    assert l.gvd_grad_sumsq(C.byref(g), None, None) == -1
    for bad in (hip.GradClip(-1.0, 1.0), hip.GradClip(float('nan'), 1.0), hip.GradClip(1.0, 0.0)):
        assert l.gvd_grad_scale(C.byref(g), C.byref(bad), a, 2, a, None) == -1
    assert l.gvd_grad_scale(C.byref(g), C.byref(c), a, 0, a, None) == -1
    g.dst_type[0] = 1                                                                        # in place, another type
    assert l.gvd_grad_scale(C.byref(g), C.byref(c), a, 2, a, None) == -1
    g.dst_type[0], g.dst[0] = 0, 0
    assert l.gvd_grad_scale(C.byref(g), C.byref(c), a, 2, a, None) == -1

    def select(**k):
        s = hip.BeamSelectArgs()
        v = dict(logits=4096, ld=50, dtype=0, B=2, K=3, V=50, W=3, eos=0, scores=4096, finished=4096, out_scores=4096, parent=4096,
                 word=4096, out_finished=4096, workspace=4096)
        v.update(k)
        for f, x in v.items():
            setattr(s, f, x)
        s.workspace_bytes = k.get('workspace_bytes', l.gvd_beam_select_workspace_bytes(s.B, s.K, s.V, s.W))
        return l.gvd_beam_select(C.byref(s), None)
    assert l.gvd_beam_select_workspace_bytes(2, 3, 50, 3) > 0
    for bad in (dict(K=33), dict(W=33), dict(W=0), dict(V=0), dict(B=0), dict(B=40000), dict(ld=49), dict(dtype=3), dict(eos=50),
                dict(eos=-2), dict(eos=-1), dict(scores=None), dict(word=None), dict(workspace=None), dict(workspace=4104),
                dict(workspace_bytes=8), dict(V=1, W=4)):
        assert select(**bad) == -1, bad

    r = hip.ReorderGroup()
    assert l.gvd_reorder_rows(C.byref(r), a, 4, 4, None) == -1
    r.count = 1
    r.t[0].src, r.t[0].dst, r.t[0].outer, r.t[0].row_bytes = 4096, 8192, 1, 8
    assert l.gvd_reorder_rows(C.byref(r), None, 4, 4, None) == -1
    assert l.gvd_reorder_rows(C.byref(r), a, 0, 4, None) == -1
    r.t[0].row_bytes = 0
    assert l.gvd_reorder_rows(C.byref(r), a, 4, 4, None) == -1
    r.t[0].row_bytes, r.t[0].outer = 1 << 40, 1 << 20
    assert l.gvd_reorder_rows(C.byref(r), a, 4, 4, None) == -1
