"""What the operators of a full-catalogue softmax model refuse, without a GPU: host tensors, wrong types and shapes in Python,
bad arguments at the C entry points (all of them are turned away before anything is launched)."""
import ctypes

import pytest
import torch


def test_python_entry_points_refuse_host_tensors():
    from mmssl_amd import ops, optim
    from mmssl_amd._lib import MmsslError
    x = torch.zeros(4, 8)
    for fn in (lambda: ops.embed_rows(x, torch.zeros(3, dtype=torch.int64)), lambda: ops.layernorm_rows(x),
               lambda: ops.logprobs_rows(x, torch.zeros(4, dtype=torch.int64)), lambda: optim.grad_norm([x]),
               lambda: optim.clip_grads([x], 1.0), lambda: optim.clip_grads([], 1.0), lambda: optim.grad_norm([]),
               lambda: optim.clip_grads([x], -1.0), lambda: optim.clip_grads([x], float("nan")),
               lambda: optim.clip_grad_norm([torch.nn.Parameter(x)], 1.0), lambda: optim.grad_norm([x.to_sparse()]),
               lambda: optim.grad_norm([x.double()])):
        with pytest.raises(MmsslError):
            fn()


BAD, UNSUPP, WORK = -1, -2, -3


def test_c_entry_points_refuse_bad_arguments():
    from mmssl_amd import _lib
    L = _lib.lib()
    p = 1 << 20                                               # an address that is never touched
    # table, ldt, dtype, rows, d, idx, idx_bytes, n, scale, has_pad, pad, out, ldo, stream
    good = [p, 8, 0, 10, 8, p, 8, 5, 1.0, 0, 0, p, 8, None]
    for at, value, code in ((0, None, BAD), (2, 3, BAD), (2, -1, BAD), (3, -1, BAD), (3, 1 << 31, UNSUPP), (4, 0, BAD),
                            (4, (1 << 24) + 1, UNSUPP), (5, None, BAD), (6, 2, BAD), (7, -1, BAD), (7, 1 << 31, UNSUPP),
                            (11, None, BAD), (12, 7, BAD), (1, -1, BAD), (0, p + 2, BAD), (5, p + 4, BAD), (11, p + 1, BAD)):
        args = list(good)
        args[at] = value
        assert L.mmssl_embed_rows(*args) == code, (at, value)
    args = list(good)
    args[7] = 0
    assert L.mmssl_embed_rows(*args) == 0                     # nothing to look up
    # g, ldg, dtype, idx, idx_bytes, n, rows, d, scale, has_pad, pad, grad, ws, ws_bytes, stream
    nb = L.mmssl_embed_rows_bwd_workspace_bytes(10, 8, 5)
    good = [p, 8, 0, p, 8, 5, 10, 8, 1.0, 0, 0, p, p, nb, None]
    for at, value, code in ((0, None, BAD), (1, -1, BAD), (2, 7, BAD), (3, None, BAD), (4, 3, BAD), (5, -1, BAD), (6, -1, BAD),
                            (7, 0, BAD), (11, None, BAD), (12, None, WORK), (12, p + 8, WORK), (13, nb - 1, WORK),
                            (6, 1 << 31, UNSUPP), (11, p + 2, BAD)):
        args = list(good)
        args[at] = value
        assert L.mmssl_embed_rows_bwd(*args) == code, (at, value)
    assert L.mmssl_embed_rows_bwd_workspace_bytes(-1, 8, 5) == 0
    # X, ldx, dtype, rows, d, w, b, pdt, eps, Y, stats, stream
    good = [p, 8, 1, 10, 8, p, p, 0, 1e-5, p, p, None]
    for at, value, code in ((0, None, BAD), (1, -8, BAD), (2, 9, BAD), (3, -1, BAD), (4, 0, BAD), (4, (1 << 24) + 1, UNSUPP),
                            (7, 3, BAD), (8, -1.0, BAD), (8, float("nan"), BAD), (9, None, BAD), (5, p + 2, BAD),
                            (0, p + 1, BAD), (10, p + 4, BAD)):
        args = list(good)
        args[at] = value
        assert L.mmssl_layernorm_rows(*args) == code, (at, value)
    nb = L.mmssl_layernorm_rows_bwd_workspace_bytes(0, 10, 8)
    # X, ldx, G, ldg, dtype, rows, d, w, pdt, stats, GX, gw, gb, ws, ws_bytes, stream
    good = [p, 8, p, 8, 0, 10, 8, p, 0, p, p, p, p, p, nb, None]
    for at, value, code in ((0, None, BAD), (2, None, BAD), (3, -1, BAD), (4, 5, BAD), (5, -1, BAD), (6, 0, BAD), (8, 4, BAD),
                            (9, None, BAD), (13, None, WORK), (14, nb - 1, WORK), (10, p + 2, BAD), (11, p + 1, BAD)):
        args = list(good)
        args[at] = value
        assert L.mmssl_layernorm_rows_bwd(*args) == code, (at, value)
    args = list(good)
    args[10] = args[11] = args[12] = None
    assert L.mmssl_layernorm_rows_bwd(*args) == 0             # no gradient is wanted
    nb = L.mmssl_logprobs_rows_workspace_bytes(0, 2, 100000, 5)
    # X, ldx, dtype, rows, cols, target, tbytes, ignore, k, T, logp, entropy, top_logp, top_idx, stats, ws, ws_bytes, stream
    good = [p, 100000, 0, 2, 100000, p, 8, -100, 5, 1.0, p, p, p, p, p, p, nb, None]
    for at, value, code in ((0, None, BAD), (1, -1, BAD), (2, 3, BAD), (3, -1, BAD), (4, 0, BAD), (4, 1 << 31, UNSUPP),
                            (5, None, BAD), (6, 1, BAD), (8, -1, BAD), (8, 129, UNSUPP), (9, 0.0, BAD), (9, -1.0, BAD),
                            (9, float("inf"), BAD), (9, float("nan"), BAD), (10, None, BAD), (11, None, BAD), (12, None, BAD),
                            (13, None, BAD), (15, None, WORK), (16, nb - 1, WORK), (3, 1 << 40, UNSUPP), (14, p + 8, BAD),
                            (13, p + 4, BAD)):
        args = list(good)
        args[at] = value
        assert L.mmssl_logprobs_rows(*args) == code, (at, value)
    args = list(good)
    args[4], args[8] = 3, 4                                   # more alternatives than columns
    assert L.mmssl_logprobs_rows(*args) == UNSUPP
    # X, ldx, dtype, rows, cols, target, tbytes, ignore, k, T, top_idx, stats, glogp, gentropy, gtop, GX, stream
    good = [p, 100, 0, 2, 100, p, 8, -100, 5, 1.0, p, p, p, p, p, p, None]
    for at, value, code in ((0, None, BAD), (2, 3, BAD), (5, None, BAD), (10, None, BAD), (11, None, BAD), (15, None, BAD),
                            (9, 0.0, BAD), (15, p + 2, BAD)):
        args = list(good)
        args[at] = value
        assert L.mmssl_logprobs_rows_bwd(*args) == code, (at, value)
    one = lambda ty, *v: (ty * len(v))(*v)      # noqa: E731
    ptrs, numel, dt = one(ctypes.c_void_p, p), one(ctypes.c_int64, 10), one(ctypes.c_int32, 0)
    nb = L.mmssl_grad_norm_workspace_bytes(1)
    good = [ptrs, numel, dt, 1, p, p, nb, None]
    for at, value, code in ((0, None, BAD), (0, one(ctypes.c_void_p, 0), BAD), (0, one(ctypes.c_void_p, p + 2), BAD),
                            (1, one(ctypes.c_int64, -1), BAD), (2, one(ctypes.c_int32, 3), BAD), (3, -1, BAD), (4, None, BAD),
                            (5, None, WORK), (6, nb - 1, WORK)):
        args = list(good)
        args[at] = value
        assert L.mmssl_grad_norm(*args) == code, (at, value)
    good = [ptrs, ptrs, numel, dt, 1, 1.0, 1e-6, p, p, nb, None]
    for at, value, code in ((1, None, BAD), (1, one(ctypes.c_void_p, 0), BAD), (5, -1.0, BAD), (5, float("nan"), BAD),
                            (6, -1.0, BAD), (7, None, BAD), (8, None, WORK), (9, nb - 1, WORK)):
        args = list(good)
        args[at] = value
        assert L.mmssl_clip_grads(*args) == code, (at, value)
    assert L.mmssl_grad_norm_workspace_bytes(-1) == 0


def test_launches_past_32_bits_of_threads_are_refused():
    from mmssl_amd import _lib
    L = _lib.lib()
    p = 1 << 20
    lp = [p, 100, 0, 1 << 24, 100, p, 8, -100, 0, 1.0, p, p, p, p, p, p, 1 << 40, None]
    assert L.mmssl_logprobs_rows(*lp) == UNSUPP
    assert L.mmssl_logprobs_rows_bwd(p, 100, 0, 1 << 24, 100, p, 8, -100, 0, 1.0, p, p, p, p, None, p, None) == UNSUPP
    assert L.mmssl_logprobs_rows_workspace_bytes(0, 1 << 24, 100, 0) == 0
    assert L.mmssl_logprobs_rows_workspace_bytes(0, (1 << 24) - 1, 100, 0) > 0
    assert L.mmssl_logprobs_rows_workspace_bytes(0, 1 << 23, 2049, 0) == 0
    assert L.mmssl_logprobs_rows_workspace_bytes(0, 1 << 62, 1, 0) == 0
    assert L.mmssl_layernorm_rows(p, 20000, 1, 1 << 22, 20000, p, p, 0, 1e-5, p, p, None) == UNSUPP
    assert L.mmssl_layernorm_rows_bwd(p, 20000, p, 20000, 1, 1 << 22, 20000, p, 0, p, p, None, None, None, 0, None) == UNSUPP
    # 16 rows a block above 64 vectors a row
    assert L.mmssl_embed_rows(p, 1000, 0, 10, 1000, p, 8, 1 << 29, 1.0, 0, 0, p, 1000, None) == UNSUPP


def test_missing_binding_fails_loudly():
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = ("import sys\nsys.modules['mmssl_amd._torch_binding'] = None\nimport torch\nfrom mmssl_amd import ops, _lib\n"
            "try:\n    ops.layernorm_rows(torch.zeros(2, 4))\nexcept _lib.MmsslError as e:\n"
            "    print('LOUD', 'no fallback' in str(e))\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True)
    assert "LOUD True" in r.stdout, r.stdout + r.stderr


def test_what_derivatives_would_lose_is_refused_before_the_device_is_looked_at():
    """Factors and gradient lists that require grad, lists with forward-mode tangents: host tensors do, the reason given is theirs."""
    from torch.autograd import forward_ad as fw
    from mmssl_amd import ops, optim
    from mmssl_amd._lib import MmsslError
    x, idx = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    two = torch.tensor(2.0, requires_grad=True)
    for fn in (lambda: ops.embed_rows(x, idx, scale=two), lambda: ops.layernorm_rows(x, eps=two * 1.0),
               lambda: ops.logprobs_rows(x, idx, temperature=two)):
        with pytest.raises(MmsslError, match="plain number"):
            fn()
    p = torch.nn.Parameter(torch.ones(4))
    for fn in (lambda: optim.grad_norm([p]), lambda: optim.clip_grads([p * 2.0], 1.0), lambda: optim.grad_norm(p)):
        with pytest.raises(MmsslError, match="not differentiable"):
            fn()
    with fw.dual_level():
        dual = fw.make_dual(torch.ones(4), torch.ones(4))
        for fn in (lambda: optim.grad_norm([dual]), lambda: optim.clip_grads([dual], 1.0)):
            with pytest.raises(MmsslError, match="forward-mode"):
                fn()
    assert bool((p == 1.0).all())


def test_factors_with_tangents_are_refused():
    from torch.autograd import forward_ad as fw
    from mmssl_amd import ops
    from mmssl_amd._lib import MmsslError
    x, idx = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    with fw.dual_level():
        two = fw.make_dual(torch.tensor(2.0), torch.tensor(1.0))
        for fn in (lambda: ops.embed_rows(x, idx, scale=two), lambda: ops.layernorm_rows(x, eps=two),
                   lambda: ops.logprobs_rows(x, idx, temperature=two)):
            with pytest.raises(MmsslError, match="plain number"):
                fn()
            with torch.no_grad(), pytest.raises(MmsslError, match="plain number"):
                fn()
    with pytest.raises(MmsslError, match="no CPU path"):          # outside the level it is a number again
        ops.embed_rows(x, idx, scale=two)
