"""The tests' generator on the host, and the kernel's, against the published vectors of Philox4x32-10."""
import numpy as np
import pytest
import torch

from tests import philox

# counter, key, numbers (Salmon, Moraes, Dror, Shaw 2011, the vectors that come with the generator)
VECTORS = [((0, 0, 0, 0), (0, 0), (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
           ((0xffffffff,) * 4, (0xffffffff,) * 2, (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
           ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0), (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1))]


def rounds(counter, key):
    """The generator, word by word."""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return tuple(c)


@pytest.mark.parametrize("counter,key,numbers", VECTORS)
def test_published_vectors(counter, key, numbers):
    assert rounds(counter, key) == numbers


@pytest.mark.parametrize("key", [0, 1, 2 ** 63 - 1, 0x299f31d0a4093822, 2 ** 64 - 1])
def test_the_host_s_numbers(key):
    counters = [0, 1, 7, 2 ** 32 - 1, 2 ** 32, 2 ** 40 + 5]
    got = philox.philox4x32(np.array(counters, dtype=np.uint64), key)
    for c, row in zip(counters, got):
        assert tuple(int(x) for x in row) == rounds((c & 0xFFFFFFFF, c >> 32, 0, 0), (key & 0xFFFFFFFF, key >> 32))


@pytest.mark.gpu
@pytest.mark.parametrize("key", [0, 1, -1, 2 ** 63 - 1, 0x299f31d0a4093822, -2 ** 63])
def test_the_kernel_s_numbers(pkg, key):
    """Ones added to zeros: an element is 1 / (1 - p) where its number is at least 65536 p, for a p between every two of
    its bits."""
    N, C = 5, 64
    zero, one = torch.zeros(N, C, device="cuda"), torch.ones(N, C, device="cuda", dtype=torch.bfloat16)
    draws = np.array([rounds((i, 0, 0, 0), (key & 0xFFFFFFFF, (key >> 32) & 0xFFFFFFFF)) for i in range(N * C // 8)], dtype=np.uint32)
    draws = torch.from_numpy(draws.astype("<u4").view("<u2").astype(np.int64)).view(N, C)
    w = torch.ones(C, device="cuda")
    for cut in (1, 3, 1000, 0x4000, 0x8000, 0xABCD, 65000, 65535):
        s, _ = pkg.residual.residual_norm(zero, one, w, w, 1e-5, dropout=cut / 65536, seed=torch.tensor([key], device="cuda"))
        want = torch.where(draws >= cut, 65536 / (65536 - cut), 0.0).float()
        assert torch.equal(s.cpu(), want), cut
