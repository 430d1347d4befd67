"""Calls whose launch would have 2^32 threads or more along one dimension: HIP runs such a launch without an error and without
the threads in excess, so the host refuses the call. Nothing is read or launched here (the pointers lead nowhere).
"""
import pytest

from fovi_amd import _lib

HERE = 4096                                              # an aligned pointer


def _refused(rc, match):
    assert rc != 0 and match in _lib.load().fovi_last_error(), _lib.load().fovi_last_error()


@pytest.mark.parametrize("dtype", [_lib.F32, _lib.BF16])
@pytest.mark.parametrize("ring", [0, 32])
@pytest.mark.parametrize("rows4", [False, True])
def test_sampler(ring, dtype, rows4):
    """2^22 views (view-major rows: 2^26, 16 to a workgroup) of 1024 points, 256 to a workgroup."""
    a = _lib.SamplerArgs()
    a.img = a.grid = a.fix_loc = a.fix_half = a.out = a.view_image = HERE
    a.img_dtype, a.out_dtype, a.mode, a.padding = dtype, dtype, _lib.BILINEAR, _lib.PAD_ZEROS
    a.n_img, a.channels, a.height, a.width, a.n_points, a.n_views, a.ring_len = 1, 3, 64, 64, 1024, 1 << 22, ring
    a.img_stride[:] = (64 * 64 * 3, 64 * 64, 64, 1)
    a.out_stride[:] = (3 * 1024, 1024, 1)
    if rows4:
        a.n_views = 1 << 26
        a.out_stride[:] = (4, 1, 4 << 26)
    _refused(_lib.load().fovi_sampler_fwd(a, None), b"exceed one launch")


def _conv(x, w, c_in, c_out):
    a = _lib.KnnConvArgs()
    a.x = a.slot_ptr = a.nbr_sorted = a.w = a.y = HERE
    a.x_dtype, a.w_dtype, a.y_dtype, a.w_layout = x, w, _lib.BF16, _lib.W_ROWS
    a.batch, a.c_in, a.n_in, a.n_out, a.k, a.n_ref, a.c_out = 1 << 24, c_in, 9, 1, 9, 9, c_out
    a.k_pad = (c_in * 9 + 63) // 64 * 64
    a.x_stride[:] = (9 * c_in, 1, c_in)
    a.y_stride[:] = (c_out, 1, c_out)
    return a


@pytest.mark.parametrize("x,c_in,c_out,match", [(_lib.F32, 16, 32, b"grid too large"), (_lib.BF16, 16, 32, b"exceed one launch"),
                                                (_lib.BF16, 64, 64, b"exceed one launch"), (_lib.BF16, 64, 256, b"exceed one launch")])
def test_kernels_of_one_image_a_workgroup(x, c_in, c_out, match):
    """kNN-conv of 2^24 images of one output point each."""
    _refused(_lib.load().fovi_knnconv_fwd(_conv(x, x, c_in, c_out), None), match)


def test_weights_and_tables():
    lib = _lib.load()
    _refused(lib.fovi_knnconv_pack_weight(HERE, 1 << 20, 64, 64, HERE, _lib.BF16, 4096, 64, None, None), b"exceed one launch")
    _refused(lib.fovi_knnconv_pack_weight_mfma(HERE, 1 << 20, 64, 64, HERE, _lib.BF16, None, None, None), b"exceed one launch")
    _refused(lib.fovi_knnconv_pack_weight_img(HERE, 1 << 20, 64, 64, HERE, _lib.BF16, None, None, HERE, None), b"too large")
    a = _lib.LocalRfArgs()
    a.src_cortical = a.src_cart = a.out_cortical = a.out_cart = a.knn_idx = a.ref = a.slots = a.flags = HERE
    a.n_src, a.dim, a.n_out, a.k, a.n_ref, a.tol = 64, 2, 1 << 26, 9, 9, 1e-3
    _refused(lib.fovi_local_rf_slots(a, None), b"n_out too large")
