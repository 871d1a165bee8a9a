"""What the training operators refuse, and the C entries' argument checks (no GPU)."""
import ctypes as C

import pytest
import torch

from hive_neuralnet_b200 import _lib, train_ops as ops


@pytest.fixture(scope="module")
def lib():
    import os
    if not os.path.exists(_lib.LIB_PATH):
        _lib.build()
    return _lib.load()


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 64)
    with pytest.raises(ValueError):
        ops.layer_norm_forward(x, torch.ones(64), torch.zeros(64))
    with pytest.raises(ValueError):
        ops.layer_norm_backward(x, x, torch.ones(64), torch.zeros(4), torch.zeros(4))
    q = torch.zeros(1, 5, 2, 8)
    at, mask = torch.zeros(1, 5, dtype=torch.int32), torch.ones(1, 5, dtype=torch.bool)
    tables = [torch.zeros(17, 2), torch.zeros(17, 2), torch.zeros(5, 2)]
    with pytest.raises(ValueError):
        ops.relative_attention_forward(q, q, q, at, at, at, mask, *tables)
    with pytest.raises(ValueError):
        ops.relative_attention_backward(q, q, q, q, at, at, at, mask, *tables, None)
    with pytest.raises(ValueError):
        ops.relative_attention_packed(q, at, at, at, mask, *tables)
    p = [torch.zeros(10)]
    with pytest.raises(ValueError):
        ops.adamw_step(p, p, torch.zeros(256), torch.zeros(256), step=1, lr=0.1)
    with pytest.raises(ValueError):
        ops.exp_avg_values(torch.zeros(256, dtype=torch.uint8), torch.zeros(1))
    with pytest.raises(ValueError):
        ops.adamw_step(p, [], torch.zeros(256), torch.zeros(256), step=1, lr=0.1)
    with pytest.raises(ValueError):
        ops.adamw_step(p, p, torch.zeros(256), torch.zeros(256), step=0, lr=0.1)
    for bad in (dict(state_bits=16), dict(lr=-1), dict(betas=(1.0, 0.9))):
        with pytest.raises(ValueError):
            ops.AdamW(p, **bad)
    with pytest.raises(ValueError):
        ops.AdamW([])
    assert ops.state_size([torch.zeros(1), torch.zeros(256), torch.zeros(257), torch.zeros(0)]) == 256 + 256 + 512


def _problem(**change):
    v = 4096
    i3, i4 = C.c_int64 * 3, C.c_int64 * 4
    a = dict(q=v, k=v, v=v, q_stride=i3(640, 64, 8), k_stride=i3(640, 64, 8), v_stride=i3(640, 64, 8), token_q=v,
             token_r=v, token_z=v, token_mask=v, token_stride=i4(10, 10, 10, 10), dq_bias=v, dr_bias=v, dz_bias=v,
             batch=2, tokens=10, queries=10, heads=8, head_dim=8, coord_clip=8, height_clip=2, dtype=0, table_dtype=0,
             scale=0.3)
    a.update(change)
    return _lib.HvAttention(**a)


@pytest.mark.parametrize("change", [
    dict(batch=-1), dict(tokens=-1), dict(queries=11), dict(queries=-1), dict(heads=0), dict(heads=70000),
    dict(head_dim=0), dict(head_dim=65), dict(coord_clip=17), dict(coord_clip=-1), dict(height_clip=5), dict(dtype=3),
    dict(dtype=1, table_dtype=2), dict(q=None), dict(v=None), dict(token_mask=None), dict(dz_bias=None)])
def test_attention_entries_refuse(lib, change):
    s = (C.c_size_t * 3)()
    at = C.addressof(s)
    a = _problem(**change)
    assert lib.hv_relative_attention_sizes(a, at, at + 8, at + 16) == 1
    assert lib.hv_relative_attention_forward(a, 4096, None, 4096, 1 << 40, None) == 1
    st = (C.c_int64 * 3)(640, 64, 8)
    sp = C.addressof(st)
    assert lib.hv_relative_attention_backward(a, 4096, sp, None, 4096, 4096, 4096, sp, sp, 4096, 4096, 4096, 4096, 1 << 40,
                                              None) == 1


def test_attention_entries_check_buffers(lib):
    a = _problem()
    assert lib.hv_relative_attention_forward(a, None, None, 4096, 1 << 40, None) == 1
    st = (C.c_int64 * 3)(640, 64, 8)
    sp = C.addressof(st)
    ok = [4096, sp, None, 4096, 4096, 4096, sp, sp, 4096, 4096, 4096, 4096, 1 << 40, None]
    for i in (0, 1, 3, 4, 5, 6, 7, 8, 9, 10):  # dout, its strides, the gradients, theirs
        bad = list(ok)
        bad[i] = None
        assert lib.hv_relative_attention_backward(a, *bad) == 1, i
    bad = list(ok)
    bad[12] = 1  # workspace too small
    assert lib.hv_relative_attention_backward(a, *bad) == 1
    bad = list(ok)
    bad[11] = 4096 + 16  # workspace off a 256-byte boundary
    assert lib.hv_relative_attention_backward(a, *bad) == 1
    assert lib.hv_relative_attention_forward(_problem(batch=0), None, None, None, 0, None) == 0


def test_norm_entries_refuse(lib):
    v = 4096
    good = [v, None, v, v, 10, 64, 0, 0, 1e-5, None, v, v, v, None]
    for i, value in ((4, -1), (5, 0), (5, 8193), (6, 3), (7, 1), (0, None), (2, None), (3, None), (10, None), (1, v),
                     (9, v), (11, None)):
        bad = list(good)
        bad[i] = value
        assert lib.hv_layer_norm_forward(*bad) == 1, i
    empty = list(good)
    empty[4] = 0
    assert lib.hv_layer_norm_forward(*empty) == 0
    need = C.c_size_t(0)
    assert lib.hv_layer_norm_workspace_bytes(10, 64, 0, C.addressof(need)) == 0 and need.value > 0
    for bad in ((-1, 64, 0), (1, 0, 0), (1, 8193, 0), (1, 64, 5)):
        assert lib.hv_layer_norm_workspace_bytes(*bad, C.addressof(need)) == 1
    good = [v, v, v, v, v, None, 10, 64, 0, 0, v, v, v, v, 1 << 30, None]
    for i, value in ((0, None), (1, None), (2, None), (3, None), (4, None), (6, -1), (7, 0), (8, 9), (9, 2), (10, None),
                     (11, None), (12, None), (13, None), (13, 4100)):
        bad = list(good)
        bad[i] = value
        assert lib.hv_layer_norm_backward(*bad) == 1, i


def test_adamw_entries_refuse(lib):
    v = 4096
    ptr, num = (C.c_void_p * 1)(v), (C.c_int64 * 1)(10)
    pa, na = C.addressof(ptr), C.addressof(num)
    good = [pa, pa, na, 1, 0, v, v, None, None, 32, .9, .1, .99, .01, 1e-8, 1., 1., 1., 0, None]
    for i, value in ((3, -1), (4, 3), (9, 16), (9, 8), (0, None), (1, None), (2, None), (5, None), (6, None), (5, 4100)):
        bad = list(good)
        bad[i] = value
        assert lib.hv_adamw_step(*bad) == 1, i
    none = list(good)
    none[3] = 0
    assert lib.hv_adamw_step(*none) == 0
    num[0] = -1
    assert lib.hv_adamw_step(*good) == 1
    num[0] = 10
    ptr[0] = 4097  # off the element's size
    assert lib.hv_adamw_step(*good) == 1
    assert lib.hv_adamw_state_values(v, v, 100, 0, v, None) == 1
    assert lib.hv_adamw_state_values(v, None, 256, 0, v, None) == 1
    assert lib.hv_adamw_state_values(None, None, 0, 0, None, None) == 0
