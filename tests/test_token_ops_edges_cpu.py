"""CPU: calls of the token-side operators that are refused before a GPU is touched, and the rules of their C entries' workspaces."""
import pytest
import torch

from gvd_amd import hip, ops


def test_reorder_refuses_a_result_over_its_index():
    """One workgroup would write the index while another still reads it."""
    words = torch.zeros(6, dtype=torch.int64)
    buf = torch.zeros(3, 6, dtype=torch.int64)
    for parent, out in ((words, words), (words.view(2, 3), words.view(-1)), (buf[1], buf[1]), (buf.view(-1)[4:10], buf[1])):
        with pytest.raises(hip.GvdHipError, match='overlaps'):
            ops.reorder_rows([torch.ones(6, dtype=torch.int64)], parent, out=[out])
    # apart from the result, or copied before the launch (its entries do not lie side by side): as far as the check of the device
    for parent in (buf[0], buf[2], buf.t()[0].repeat(2), buf.t()[:2].reshape(-1)):
        with pytest.raises(hip.GvdHipError, match='no CPU fallback'):
            ops.reorder_rows([torch.ones(6, dtype=torch.int64)], parent, out=[buf[1]])


def test_embedding_refuses_a_table_with_a_tangent():
    """There is no forward-mode rule: a tangent is refused, not lost, whether or not the table requires a gradient too."""
    import torch.autograd.forward_ad as fw
    tok, w = torch.zeros(3, dtype=torch.int64), torch.randn(7, 4)
    with fw.dual_level():
        for grad in (False, True):
            dual = fw.make_dual(w.clone().requires_grad_(grad), torch.ones(7, 4))
            for table in (dual, dual[:, 1:3], dual.t().contiguous().t()):
                with pytest.raises(hip.GvdHipError, match='forward-mode'):
                    ops.embedding(tok, table)
        with pytest.raises(hip.GvdHipError, match='no CPU fallback'):
            ops.embedding(tok, w)                   # no tangent: as far as the check of the device
    with pytest.raises(hip.GvdHipError, match='forward-mode'):
        torch.func.jvp(lambda t: ops.embedding(tok, t), (w,), (w,))


def test_embedding_workspace_is_what_the_function_says():
    """Few tokens alone do not make it 0: with a large table the gradient is refused without it, before anything is launched."""
    import ctypes as C
    l, a = hip.lib(), C.c_void_p(4096)
    for n, vocab, width in ((1, 70001, 129), (4096, 50000, 1024)):
        need = l.gvd_embedding_bwd_workspace_bytes(n, vocab, width)
        assert need > 0
        for ws, size in ((None, need), (a, need - 1), (None, 0)):
            assert l.gvd_embedding_bwd(a, 1, n, a, width, a, width, vocab, width, 0, 1.0, 0, -1, a, ws, size, None) == -1
    assert l.gvd_embedding_bwd_workspace_bytes(4096, 5000, 512) == 0 == l.gvd_embedding_bwd_workspace_bytes(1, 1, 1)


def test_embedding_one_launch_is_for_tables_of_few_workgroups():
    """Every workgroup of the one-launch gradient looks at all tokens, so it is for tables of at most 512 of them (64 rows x 256
    columns, or a narrower table's whole width): narrow tables of many rows are sorted for."""
    need = hip.lib().gvd_embedding_bwd_workspace_bytes
    for n in (5, 4096):
        for vocab, width in ((32768, 32), (32768, 256), (32768, 1), (16384, 512), (8192, 1024), (5000, 512), (64, 1 << 17)):
            assert need(n, vocab, width) == 0, (n, vocab, width)
        for vocab, width in ((32769, 32), (131072, 32), (1 << 20, 8), (1 << 23, 1), (27000, 300), (32768, 257), (65, 1 << 17)):
            assert need(n, vocab, width) > 0, (n, vocab, width)
