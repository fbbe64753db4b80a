"""Sizes at which an MXFP4 call passes what one launch holds, 2^32 threads (CPU): refused
with an error, or run on a larger tile."""
import pytest

import mx_plans
from acfun_amd import capi

FAR = [(i + 1) << 44 for i in range(8)]      # stand for device addresses; never read
TOO = "too large"


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    exe = mx_plans.build(tmp_path_factory.mktemp("mx_plan"))
    return lambda *lines: mx_plans.ask(exe, lines)


def _refused(rc):
    assert rc == -1 and TOO in capi.last_error(), (rc, capi.last_error())


def test_quantizer():
    """2^28 rows of one scale tile are 2^24 workgroups of 256 threads."""
    L = capi.lib()
    for rows, K, trans in ((1 << 28, 32, 0), (1 << 28, 512, 1), (1 << 27, 513, 0), ((1 << 28) - 15, 1, 0),
                           ((1 << 31) - 1, 1, 1), (1 << 20, 1 << 20, 0)):
        for t in range(3):
            _refused(L.acfun_dev_quantize_mxfp4(FAR[0], t, rows, K, trans, FAR[1], FAR[2], None))
            if not trans:
                _refused(L.acfun_dev_dequantize_mxfp4(FAR[1], FAR[2], rows, K, FAR[0], t, None))


def test_quantizer_edge(plans):
    last = (1 << 28) - 16                    # 2^24 - 1 tiles of 16 rows
    assert plans(f"quant {last} 32 0", f"quant {last + 1} 32 0", f"quant {last - 64} 32 1",
                 f"quant {1 << 28} 32 1") == ["fits", "not", "fits", "not"]


def test_products_refused():
    L = capi.lib()
    for M, N, K in (((1 << 31) - 1, 1 << 18, 32), (1 << 20, 1 << 20, 64), (1 << 19, 1 << 18, 0),
                    (1 << 18, 1 << 18, (1 << 22) + 1)):
        _refused(L.acfun_dev_gemm_mxfp4(M, N, K, FAR[0], FAR[1], FAR[2], FAR[3], FAR[4], 1, None, 0, None))
        _refused(L.acfun_dev_fc_mxfp4(FAR[0], 1, M, K, FAR[2], FAR[3], None, N, FAR[4], 0, None))


def test_layers_refused():
    """Rows of which neither the quantizer's launch nor one launch of 16 rows each can have so many."""
    L = capi.lib()
    _refused(L.acfun_dev_fc_mxfp4(FAR[0], 1, 1 << 28, 64, FAR[2], FAR[3], None, 16, FAR[4], 0, None))


@pytest.mark.parametrize("M,N,K,want", [
    # tiles of 32 are the fastest here while their launch holds the call; those of 64 hold no more
    (1, (1 << 29) - 512, 700, "FEW32"), (1, 1 << 29, 700, "MANY128"), (1, (1 << 31) - 1, 500, "MANY256"),
    # the largest launch of the largest tile, and one more tile row
    ((1 << 20) - 2048, 1 << 20, 4096, "MANY256"), (1 << 20, 1 << 20, 4096, "none"),
    # K = 0 and K past MANY's offsets have tiles of 64 at most
    (1 << 18, (1 << 17) - 512, 0, "FEW64"), (1 << 18, 1 << 17, 0, "none"),
    ((1 << 31) - 1, (1 << 31) - 1, (1 << 31) - 1, "none")])
def test_larger_tiles(plans, M, N, K, want):
    """Each tile only where its launch holds the call (the program checks that it is one
    that mm_fits says is there)."""
    got = plans(mx_plans.gemm(M, N, K))[0]
    assert got == want
    if got != "none":
        edge, threads = {"FEW16": (16, 512), "FEW32": (32, 256), "FEW64": (64, 512), "MANY128": (128, 256),
                         "MANY256": (256, 256)}[got]
        assert (-(-M // edge) * -(-N // edge) + 7) // 8 * 8 * threads < 1 << 32


def test_every_tile_fits(plans):
    """Over sizes of every magnitude: the tile taken holds the call."""
    sizes = [(M, N, K) for M in (1, 100, 5000, 1 << 17, 1 << 24) for N in (16, 5000, 1 << 20, 1 << 27, (1 << 31) - 1)
             for K in (1, 500, 8192, 1 << 20, (1 << 22) + 1)]
    edges = {"FEW16": (16, 512), "FEW32": (32, 256), "FEW64": (64, 512), "MANY128": (128, 256), "MANY256": (256, 256)}
    for (M, N, K), got in zip(sizes, plans(*(mx_plans.gemm(*s) for s in sizes))):
        fits = [n for n, (e, t) in edges.items()
                if (-(-M // e) * -(-N // e) + 7) // 8 * 8 * t < 1 << 32 and (n[0] == "F" or K <= 1 << 22)]
        assert got in fits or (got == "none" and not fits), (M, N, K)
