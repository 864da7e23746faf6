"""The C entries of the adapter operators at the edges of what they accept, called as a host without Python would."""
import pytest
import torch

from aqualora_amd import _lib as L

DEV = "cuda"
gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("M", [65536, 40000])
def test_weight_rows_far_apart(M):
    """Rows of W at the largest leading dimension: 320 of them reach past 1 GiB.  Small whole numbers, so the products are exact."""
    N, K, ldw = 320, 8, (1 << 21) - 8
    gen = torch.Generator().manual_seed(1)
    x = torch.randint(-3, 4, (M, K), generator=gen).to(DEV, torch.bfloat16)
    w = torch.empty(N, ldw, dtype=torch.bfloat16, device=DEV)
    w[:, :K] = torch.randint(-3, 4, (N, K), generator=gen).to(DEV, torch.bfloat16)
    y = torch.full((M, N), float("nan"), dtype=torch.bfloat16, device=DEV)
    L.call("aql_adapter_linear", L.ptr(x), K, L.ptr(w), ldw, None, None, 0, L.ptr(y), N, M, N, K, None, None, None, None, 0, None, 1, 0, 1, 0, None, 1, L.stream_ptr())
    assert torch.equal(y.float(), x.float() @ w[:, :K].float().t())


def test_stacks_of_ranks_beyond_the_descriptors_are_refused():
    lib = L.load()
    p = L.c_p(4096)     # never dereferenced: the calls are refused on the host
    linear = lambda R, parts: lib.aql_adapter_linear(p, 64, p, 64, None, None, 0, p, 64, 300, 64, 64, p, p, p, p, R, p, 1, 1, 1, 1, p, parts, None)  # noqa: E731
    down = lambda R: lib.aql_adapter_down(p, 64, None, None, 300, 64, p, p, p, R, p, 1, 1, 1, p, 3, None)  # noqa: E731
    for R in ((1 << 16) + 8, 1 << 20, 1 << 30):
        assert linear(R, 1) != 0 and linear(R, 3) != 0 and b"R=" in lib.aql_last_error()
        assert down(R) != 0
