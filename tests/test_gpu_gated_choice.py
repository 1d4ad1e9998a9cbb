"""Which kernel a forward call goes to.  All tiles sum over K in the same order, the blocks of few
tokens in another one, so the bits tell them apart; the sizes are on both sides of the
border, where the times beside the rule differ by more than the 8% that it may miss."""
import pytest
import torch

from test_gpu_gated import _close, _want

pytestmark = pytest.mark.gpu


def _bits(et, dev, T, K, F):
    """(the call's result, every kind of tiles')"""
    g = torch.Generator(device=dev).manual_seed(T + K + F)
    x = torch.randn(T, K, generator=g, device=dev).bfloat16()
    w = (torch.randn(2 * F, K, generator=g, device=dev) * K ** -0.5).bfloat16()
    tiles = []
    for kind in (2, 4, 6, 8):
        h = torch.empty(T, F, device=dev, dtype=torch.bfloat16)
        assert et.lib().et_gated_linear_impl(x.data_ptr(), K, w.data_ptr(), T, K, F, 0, h.data_ptr(), kind,
                                             torch.cuda.current_stream().cuda_stream) == 0
        tiles.append(h)
    assert all(torch.equal(t, tiles[0]) for t in tiles)
    got = et.gated_linear(x, w)
    _close(got, _want(x, w, "silu")["h"], "h")
    return got, tiles[0]


@pytest.mark.parametrize("T,K,F", [(6000, 512, 64), (4096, 7168, 64), (192, 512, 2048), (768, 512, 512), (384, 1024, 1024),
                                   (8, 512, 8192), (256, 4096, 2048), (1536, 1024, 256)])
def test_tiles(et, dev, T, K, F):
    got, tiles = _bits(et, dev, T, K, F)
    assert torch.equal(got, tiles)


@pytest.mark.parametrize("T,K,F", [(1, 4096, 2048), (64, 512, 2048), (61, 2048, 1408), (1024, 2048, 256), (2048, 7168, 64),
                                   (192, 4096, 2048), (17, 7168, 8192), (32, 4096, 8192)])
def test_few_tokens(et, dev, T, K, F):
    got, tiles = _bits(et, dev, T, K, F)
    assert not torch.equal(got, tiles)
