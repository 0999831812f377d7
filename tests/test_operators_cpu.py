"""What the operators in three types refuse before anything reaches the GPU, and their workspace sizes."""
import ctypes

import pytest
import torch

from focalformer3d_amd import _lib, ops, training


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(3, 8), torch.zeros(4, 8)
    for call in (lambda: ops.gated_linear(x, w), lambda: ops.gated_linear_bwd(x, w, None, 'silu', torch.zeros(3, 2)), lambda: ops.grad_norm([x]),
                 lambda: ops.diff_attention(torch.zeros(1, 3, 32), torch.zeros(1, 3, 32), torch.zeros(1, 3, 32), torch.zeros(1), 1),
                 lambda: ops.clip_grads([x], 1.0), lambda: training.clip_grads([], 1.0)):
        with pytest.raises(RuntimeError, match='CUDA'):
            call()


def test_no_gradients_have_norm_zero():
    p = torch.nn.Parameter(torch.zeros(3))
    assert float(training.clip_grad_norm_([p], 1.0)) == 0.0


def test_norm_kinds():
    with pytest.raises(ValueError):
        ops._norm_kind(3)
    assert [ops._norm_kind(k) for k in (2, 1.0, float('inf'))] == [2, 1, 0]


def test_dense_layouts():
    t = torch.zeros(4, 6, 5)
    assert ops._dense(t) and ops._dense(t.permute(2, 0, 1)) and ops._dense(t[1:3]) and ops._dense(torch.zeros(3, 1, 4).transpose(0, 1))
    assert not ops._dense(t[:, ::2]) and not ops._dense(t[:, 1:3]) and not ops._dense(torch.zeros(1).expand(4))


def test_c_entries_check_their_arguments():
    """Every refusal returns its status without touching a pointer: the addresses here are none."""
    lib = _lib.load()
    f = lib.ff3d_gated_linear_fwd
    p = ctypes.c_void_p(4096)
    ok = dict(x=p, ldx=16, w=p, b=None, h=p, M=2, C=16, F=4, act=0, dt=0, pack=0, ws=None)
    run = lambda **k: f(*{**ok, **k}.values(), None)  # noqa: E731
    assert run(x=None) == -4 and run(w=None) == -4 and run(h=None) == -4
    assert run(dt=2) == -2 and run(dt=7) == -2
    for bad in (dict(M=0), dict(M=0x7fffff00), dict(C=0), dict(F=-1), dict(ldx=15), dict(act=4), dict(pack=4), dict(C=1 << 20, F=1 << 20, ldx=1 << 20)):
        assert run(**bad) == -1, bad
    assert run(ldx=17) == -3 and run(x=ctypes.c_void_p(4100)) == -3 and run(w=ctypes.c_void_p(4104)) == -3
    assert run(C=15) == -3 and run(C=15, pack=1) == -3
    assert run(C=15, pack=3) == -4 and run(C=15, pack=3, ws=ctypes.c_void_p(4100)) == -3          # needs a workspace
    assert lib.ff3d_gated_linear_workspace_bytes(2, 16, 4, 0, 0, 0) == 0
    # packed rows of 16 floats, each part on 256 bytes
    assert lib.ff3d_gated_linear_workspace_bytes(2, 15, 4, 0, 3, 0) == 256 + 512
    norm = lib.ff3d_grad_norm
    ptrs, numel, code = (ctypes.c_void_p * 1)(4096), (ctypes.c_int64 * 1)(5), (ctypes.c_int32 * 1)(0)
    assert norm(ptrs, numel, code, 1, 3, p, p, None) == -1 and norm(ptrs, (ctypes.c_int64 * 1)(-1), code, 1, 2, p, p, None) == -1
    assert norm(ptrs, numel, (ctypes.c_int32 * 1)(2), 1, 2, p, p, None) == -2
    assert norm((ctypes.c_void_p * 1)(None), numel, code, 1, 2, p, p, None) == -4 and norm(ptrs, numel, code, 1, 2, None, p, None) == -4
    clip = lib.ff3d_clip_grads
    two, n2, c2 = (ctypes.c_void_p * 2)(4096, 4096 + 12), (ctypes.c_int64 * 2)(5, 5), (ctypes.c_int32 * 2)(0, 0)
    assert clip(two, two, n2, c2, c2, 2, 2, 1.0, p, p, None) == -5
    assert clip(ptrs, None, numel, code, code, 1, 2, 1.0, p, p, None) == -4
    # four elements, one piece, one more for none
    assert lib.ff3d_grad_norm_workspace_bytes((ctypes.c_int64 * 2)(4, 0), 2) == 16


def test_diff_attention_entry_checks_its_arguments():
    lib = _lib.load()
    P = 4096
    ok = dict(q=P, k=P, v=P, lam=P, mask=None, kv_lens=None, q_batch=320, q_row=64, k_batch=320, k_row=64, v_batch=320, v_row=64, mask_batch=0, mask_row=0,
              B=2, Nq=5, Nk=5, heads=2, kv_heads=2, d=16, causal=0, dtype=0, scale=0.25)

    def run(out=P, out2=None, lse=None, rest=None, ws=None, **k):
        return lib.ff3d_diff_attention_fwd(_lib.DiffAttention(**{**ok, **k}), out, out2, lse, rest, ws, None)
    assert lib.ff3d_diff_attention_fwd(None, P, None, None, None, None, None) == -4
    for n in ('q', 'k', 'v', 'lam', 'out'):
        assert run(**{n: None}) == -4, n
    assert run(out2=P) == -4 and run(lse=P) == -4 and run(out2=P, lse=P, dtype=1) == -4 and run(rest=P, dtype=1) == -4
    assert run(dtype=2) == -2 and run(d=24) == -5
    for bad in (dict(B=0), dict(Nq=0), dict(Nk=-1), dict(heads=3), dict(kv_heads=0), dict(scale=0.0), dict(scale=float('nan')), dict(q_row=60), dict(k_row=32),
                dict(q_batch=-320), dict(mask_row=-1), dict(Nk=1 << 30), dict(q_row=1 << 22)):
        assert run(**bad) == -1, bad
    for bad in (dict(q=P + 4), dict(q_row=66), dict(v_batch=322), dict(out=P + 8)):
        assert run(**bad) == -3, bad
    # few rows over long keys need a place for the slices
    assert run(Nq=1, Nk=2048, heads=2) == -4
    p = _lib.DiffAttention(**{**ok, 'Nq': 1, 'Nk': 2048})
    assert lib.ff3d_diff_attention_workspace_bytes(p, 0) == 4 * 4 * 1 * (4 * 16 + 4) * 4          # 4 slices of 512 keys, 4 rows
    assert lib.ff3d_diff_attention_workspace_bytes(_lib.DiffAttention(**ok), 0) == 0
    assert lib.ff3d_diff_attention_workspace_bytes(_lib.DiffAttention(**ok), 1) == 4 * (6 + 1) * 64 * 4  # rows rounded up to 64

    def bwd(out=P, out2=P, lse=P, rest=None, dout=P, db=320, dr=64, dq=P, dk=P, dv=P, dlam=P, ws=P, **k):
        return lib.ff3d_diff_attention_bwd(_lib.DiffAttention(**{**ok, **k}), out, out2, lse, rest, dout, db, dr, dq, dk, dv, dlam, ws, None)
    for n in ('out', 'out2', 'lse', 'dout', 'ws', 'dk', 'dv'):
        assert bwd(**{n: None}) == -4, n
    assert bwd(dtype=1) == -4
    assert bwd(dr=32) == -1 and bwd(dr=66) == -3 and bwd(dq=P + 4) == -3


def test_modules_refuse_what_they_cannot_do():
    import focalformer3d_amd.transformer  # noqa: F401
    from focalformer3d_amd.registry import build_attention, build_feedforward_network
    ok = dict(type='DifferentialAttention', embed_dims=64, num_heads=4)
    m = build_attention(dict(ok, dropout=0.1, batch_first=True))
    assert m.kv_heads == 4 and m.dropout_layer.p == 0.1 and tuple(m.lam().shape) == (4,)
    assert tuple(build_attention(dict(ok, kv_heads=2)).k_proj.weight.shape) == (32, 64)
    for bad in (dict(num_heads=3), dict(num_heads=8), dict(embed_dims=60), dict(kv_heads=3), dict(kv_heads=0), dict(embed_dims=1024)):
        with pytest.raises(ValueError):
            build_attention({**ok, **bad})
    for bad in (dict(attn_drop=0.1), dict(dropout_layer=dict(type='DropPath', drop_prob=0.1))):
        with pytest.raises(NotImplementedError):
            build_attention({**ok, **bad})
    x = torch.zeros(2, 5, 64)
    for bad in (dict(key=x.clone()), dict(value=x.clone()), dict(identity=x), dict(query_pos=x, key_pos=x.clone())):
        with pytest.raises(NotImplementedError):
            m(x, **bad)
    with pytest.raises(RuntimeError, match='CUDA'):
        m(x)
    ffn = dict(type='GatedFFN', embed_dims=64, feedforward_channels=96)
    g = build_feedforward_network(ffn)
    assert tuple(g.in_proj.weight.shape) == (192, 64) and g.act == 'silu'
    for bad in (dict(num_fcs=3), dict(act_cfg=dict(type='Tanh')), dict(dropout_layer=dict(type='Dropout', drop_prob=0.5))):
        with pytest.raises(NotImplementedError):
            build_feedforward_network({**ffn, **bad})
    with pytest.raises(RuntimeError, match='CUDA'):
        g(x)
