"""What the C entry points of the dense operators refuse, without a GPU: nothing is launched for a bad argument."""
import ctypes as C

import pytest

from tile_fusion_b200 import _lib

P = 4096  # an address that is never followed


@pytest.fixture(scope="module")
def L(built_lib):
    return _lib.lib()


def refused(rc, word=""):
    assert rc in (_lib.TF_ERR_ARG, _lib.TF_ERR_UNSUPPORTED)
    assert word in _lib.lib().tf_last_error().decode()


def test_layer_norm(L):
    fwd = lambda **k: L.tf_layer_norm_fwd(*{**dict(x=P, ld=8, t=0, w=None, b=None, wt=0, n=4, d=8, eps=1e-5, y=P, ldy=8, m=None, r=None, c=None, ldc=0, e=None, s=None), **k}.values())  # noqa: E731
    refused(fwd(t=3), "type")
    refused(fwd(wt=-1), "type")
    refused(fwd(n=-1), "size")
    refused(fwd(d=0), "size")
    refused(fwd(d=16385, ld=20000, ldy=20000), "columns")
    refused(fwd(x=None), "null")
    refused(fwd(ld=7), "overlap")
    refused(fwd(c=P, ldc=8, e=P), "codes")
    refused(fwd(c=P + 1, ldc=32, e=P), "codes")
    refused(fwd(c=P, ldc=32, e=None), "codes")
    assert fwd(n=0, x=None, y=None) == 0
    bwd = lambda **k: L.tf_layer_norm_bwd(*{**dict(x=P, ld=8, c=None, ldc=0, e=None, t=0, w=None, wt=0, n=4, d=8, m=P, r=P, dy=P, ldy=8, dx=P, ldx=8, dw=P, db=P, work=P, wn=1 << 20, s=None), **k}.values())  # noqa: E731
    refused(bwd(m=None), "null")
    refused(bwd(work=None), "null")
    refused(bwd(wn=2 * 8 * 4 - 1), "work")
    refused(bwd(ldx=4), "overlap")
    refused(bwd(x=None), "null")
    assert L.tf_layer_norm_work_floats(4, 8) == 64 and L.tf_layer_norm_work_floats(-1, 8) == 0


def test_pack8(L):
    pack = lambda **k: L.tf_pack8(*{**dict(x=P, ld=40, t=0, n=4, d=40, relu=0, c=P, ldc=64, e=P, s=None), **k}.values())  # noqa: E731
    refused(pack(t=9), "type")
    refused(pack(d=0), "size")
    refused(pack(ld=39), "overlap")
    refused(pack(ldc=40), "groups")
    refused(pack(ldc=32), "overlap")
    refused(pack(c=P + 16), "alignment")
    refused(pack(e=None), "null")
    assert pack(n=0) == 0
    refused(L.tf_unpack8(P, 64, None, 0, 4, 40, P, 40, None), "null")
    refused(L.tf_relu_grad8(P, 64, 0, 4, 40, None, 40, None), "null")
    grad = lambda **k: L.tf_weight_grad8(*{**dict(g=P, ld=8, t=0, na=8, c=P, ldc=64, e=P, nb=40, m=4, out=P, work=P, wn=1 << 20, s=None), **k}.values())  # noqa: E731
    refused(grad(g=None), "null")
    refused(grad(ld=7), "overlap")
    refused(grad(ldc=48), "groups")
    refused(grad(wn=1), "work")
    refused(grad(work=P + 4), "aligned")
    refused(grad(na=1 << 14, ld=1 << 14, nb=1 << 13, ldc=1 << 13), "entries")
    assert L.tf_weight_grad8_work_floats(0, 8, 40, 0) >= 8 * 40


def test_linear_ce(L):
    need = L.tf_linear_ce_work_bytes(4, 8, 5, 0, 0)
    fwd = lambda **k: L.tf_linear_ce_fwd(*{**dict(x=P, ldx=8, w=P, ldw=8, t=0, y=P, n=4, d=8, v=5, ig=-100, red=1, loss=P, lse=P, work=P, wn=need, s=None), **k}.values())  # noqa: E731
    refused(fwd(t=5), "type")
    refused(fwd(v=0), "size")
    refused(fwd(y=None), "null")
    refused(fwd(ldw=7), "overlap")
    refused(fwd(red=3), "reduction")
    refused(fwd(work=P + 16), "aligned")
    refused(fwd(wn=need - 1), "work")
    refused(fwd(loss=None), "null")
    need = L.tf_linear_ce_work_bytes(4, 8, 5, 0, 1)
    bwd = lambda **k: L.tf_linear_ce_bwd(*{**dict(x=P, ldx=8, w=P, ldw=8, t=0, y=P, n=4, d=8, v=5, ig=-100, red=1, lse=P, g=P, dx=P, dw=P, work=P, wn=need, s=None), **k}.values())  # noqa: E731
    refused(bwd(lse=None), "null")
    refused(bwd(g=None), "null")
    refused(bwd(wn=need - 1), "work")
    assert bwd(dx=None, dw=None) == 0
    refused(L.tf_linear_ce_status(None, None), "null")
    # the slope of a large vocabulary is held in pieces: 8 192 rows of 128 000 classes in bf16 are 2 GB, a piece 256 MB
    big = L.tf_linear_ce_work_bytes(8192, 4096, 128_000, 1, 1)
    assert C.c_longlong(big).value < 8192 * 128_000 * 2 / 2 + 3 * 128_000 * 4096


def test_weight_grad8_of_a_very_long_side(L):
    """A side of more than 2^20 would overflow a slice's count of bytes and the grid."""
    grad = lambda **k: L.tf_weight_grad8(*{**dict(g=P, ld=8, t=0, na=8, c=P, ldc=64, e=P, nb=40, m=4, out=P, work=P, wn=1 << 40, s=None), **k}.values())  # noqa: E731
    refused(grad(na=1 << 26, ld=1 << 26, nb=1, ldc=32), "side")
    refused(grad(na=(1 << 20) + 1, ld=(1 << 20) + 1, nb=1, ldc=32), "side")
    refused(grad(na=1, ld=1, nb=(1 << 20) + 1, ldc=(1 << 20) + 32), "side")


def test_rows_next_to_2_31(L):
    """A row's index and a step of the grid beyond it must fit 32 bits."""
    n = 0x7f000001
    refused(L.tf_layer_norm_fwd(P, 8, 0, None, None, 0, n, 8, 1e-5, P, 8, None, None, None, 0, None, None), "size")
    refused(L.tf_layer_norm_bwd(P, 8, None, 0, None, 0, None, 0, n, 8, P, P, P, 8, P, 8, None, None, None, 0, None), "size")
    refused(L.tf_pack8(P, 8, 0, n, 8, 0, P, 32, P, None), "size")
    refused(L.tf_weight_grad8(P, 8, 0, 8, P, 32, P, 8, n, P, P, 1 << 40, None), "size")
    refused(L.tf_linear_ce_fwd(P, 8, P, 8, 0, P, n, 8, 5, -100, 1, P, P, P, 1 << 40, None), "size")
    refused(L.tf_linear_ce_fwd(P, 8, P, 8, 0, P, 4, 8, n, -100, 1, P, P, P, 1 << 40, None), "size")
    assert L.tf_linear_ce_work_bytes(n, 8, 5, 0, 0) == 0 and L.tf_weight_grad8_work_floats(n, 8, 8, 0) == 0


def test_layer_that_keeps_8_bits_refuses(built_lib):
    import torch
    from tile_fusion_b200 import sw_gcn  # noqa: F401
    ck8 = torch.ops.sw_gcn.fusedGeMMSpMM_ck8
    i = torch.arange(5, dtype=torch.int32)
    adj = torch.sparse_csr_tensor(i, i[:4], torch.ones(4), size=(4, 4))
    with pytest.raises(ValueError, match="CUDA"):
        ck8(adj, torch.ones(4, 8), torch.ones(2, 8), [], 1)
    with pytest.raises(ValueError, match="chain"):
        ck8(adj, torch.ones(4, 8), torch.ones(2, 7), [], 1)
    wide = torch.sparse_csr_tensor(i[:4], i[:3], torch.ones(3), size=(3, 4))  # its gradient would read rows that are not there
    with pytest.raises(ValueError, match="square"):
        ck8(wide, torch.ones(4, 8), torch.ones(2, 8), [], 1)


def test_8_bits_of_no_matrix(built_lib):
    import torch
    from tile_fusion_b200 import sw_gcn  # noqa: F401
    with pytest.raises(ValueError, match="codes"):
        torch.ops.sw_gcn.unpack8(torch.zeros((), dtype=torch.int8), torch.zeros(1, dtype=torch.uint8))


def test_wait_limit(L):
    for polls in (-1, 1, 65535):
        refused(L.tf_dense_set_wait_limit(polls), "polls")
    assert L.tf_dense_set_wait_limit(65536) == 0 and L.tf_dense_set_wait_limit(0) == 0 and L.tf_dense_set_wait_limit(1 << 22) == 0


def test_weight_grad8_of_rows_far_apart(L):
    """16 rows of codes more than 2^26 bytes apart overflow the 32 bits that a slice's bytes are counted in; and no work space for what is refused."""
    grad = lambda **k: L.tf_weight_grad8(*{**dict(g=P, ld=8, t=0, na=8, c=P, ldc=64, e=P, nb=40, m=4, out=P, work=P, wn=1 << 40, s=None), **k}.values())  # noqa: E731
    for ld in ((1 << 26) + 32, 1 << 27, 1 << 28, 0x7fffffe0):
        refused(grad(ldc=ld), "apart")
    assert L.tf_weight_grad8_work_floats(10, 1 << 20, 1 << 20, 0) == 0 and L.tf_weight_grad8_work_floats(10, (1 << 20) + 1, 1, 1) == 0
    assert L.tf_weight_grad8_work_floats(10, 1 << 13, 1 << 13, 1) == 1 << 26


@pytest.mark.parametrize("dtype", [_lib.BF16, _lib.F16])
def test_work_space_of_a_loss(L, dtype):
    """Operands that are multiplied as they lie need no copy: 8 192 x 4 096 with 128 000 classes took 1 GB for one of the weights."""
    n, d, v = 8192, 4096, 128_000
    size = lambda x, ldx, w, ldw, back: L.tf_linear_ce_work_bytes_for(x, ldx, w, ldw, n, d, v, dtype, back)  # noqa: E731
    weights, rows = 2 * v * d, 2 * n * d
    for back in (0, 1):
        most = L.tf_linear_ce_work_bytes(n, d, v, dtype, back)
        assert size(P + 2, d, P + 2, d, back) == size(P, d + 4, P, d + 4, back) == most
        assert most - size(P + 2, d, P, d, back) == weights
        assert most - size(P, d, P + 2, d, back) == (0 if back else rows)  # (the backward pass clears rows that do not count in a copy)
    assert size(P, d, P, d, 0) < weights // 8
    assert size(P, d, P, d, 1) < 2 * rows + (600 << 20)
    assert L.tf_linear_ce_work_bytes_for(P, d, P, d, n, d, v, _lib.F32, 0) == L.tf_linear_ce_work_bytes(n, d, v, _lib.F32, 0)
    fwd = lambda need: L.tf_linear_ce_fwd(P, 64, P, 64, dtype, P, 4, 64, 300, -100, 1, P, P, P, need, None)  # noqa: E731
    need = L.tf_linear_ce_work_bytes_for(P, 64, P, 64, 4, 64, 300, dtype, 0)
    refused(fwd(need - 1), "work")
    assert L.tf_linear_ce_work_bytes_for(P, 64, P, 64, 0x7f000001, 64, 300, dtype, 0) == 0


def test_work_space_of_a_weight_gradient(L):
    """Of the result's size where that is large, however many rows: a million rows of 16-bit gradients for 2^26 entries took 31 times as much."""
    for dtype in (_lib.F32, _lib.BF16, _lib.F16):
        for m in (1, 100_000, 1_000_000, 0x7f000000):
            assert L.tf_weight_grad8_work_floats(m, 1 << 13, 1 << 13, dtype) <= 2 << 26
            assert L.tf_weight_grad8_work_floats(m, 47, 256, dtype) <= (64 << 20) + 2 * 47 * 256
            assert L.tf_weight_grad8_work_floats(m, 1000, 700, dtype) <= (64 << 20) + 2 * 1000 * 700
    assert L.tf_weight_grad8_work_floats(1_000_000, 256, 100, _lib.BF16) == 148 * 256 * 100


def test_ranges_of_very_many_rows(L):
    """A range's rows on top of 2^31 - 2^24 pass 32 bits: 16 ranges for 9 tiles became one, of a sixteenth of the rows."""
    assert L.tf_weight_grad8_work_floats(0x7f000000, 300, 600, _lib.F32) == 16 * 300 * 600
    assert L.tf_weight_grad8_work_floats(0x7f000000, 300, 300, _lib.F32) == 148 // 6 * 300 * 300
