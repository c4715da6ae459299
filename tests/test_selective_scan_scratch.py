"""The memory that the selective scan's backward asks for (no GPU: the library's own answers)."""
import pytest

from subq_audio import _capi

FAKE = 1 << 40
GIB = 1 << 30


def tensor(at, *strides):
    return _capi.Tensor3(at, *strides)


def backward_bytes(B, L, D, N, G=1, handover=True):
    """Workspace of a backward with a handover, from arguments whose tensors lie far apart."""
    a = _capi.SelectiveBwdArgs()
    d = a.desc
    d.batch, d.seq_len, d.channels, d.states, d.groups, d.dtype, d.softplus, d.A = B, L, D, N, G, 0, 1, FAKE
    for i, name in enumerate(("u", "dt", "dout", "du", "ddt")):
        setattr(a, name, tensor(FAKE * (i + 2), L * D, D, 0))
    for i, name in enumerate(("B", "C", "dB", "dC")):
        setattr(a, name, tensor(FAKE * (i + 8), L * G * N, G * N, N))
    a.dA = FAKE * 13
    if handover:
        a.handover = FAKE * 14
    return _capi.selective_scan_bwd_workspace_bytes(a), _capi.selective_scan_handover_bytes(d)


@pytest.mark.parametrize("B,L,D,N,G", [(1, 65536, 1536, 128, 1), (1, 65536, 1536, 64, 1), (4, 4096, 4096, 128, 1), (16, 1024, 1536, 100, 2),
                                       (1, 1 << 20, 64, 128, 1), (3, 50001, 1000, 40, 4), (1, 65536, 1536, 16, 1), (64, 2048, 2048, 128, 8)])
def test_parts_of_dB_and_dC_are_bounded(B, L, D, N, G):
    n = 16 if N <= 16 else 32 if N <= 32 else 64 if N <= 64 else 128
    need, kept = backward_bytes(B, L, D, N, G)
    # the parts; what the segments (256 at most) and the sums over tokens keep: three times a state of each
    states = (B * 256 * D * n * 4 + 256) * 3
    assert 0 < need <= max(GIB, 4 * B * L * D) + 256 + min(states, need)
    assert kept == (B * ((L + 7) // 8) * D * n * 4 + 255) // 256 * 256
    without, _ = backward_bytes(B, L, D, N, G, handover=False)
    assert kept < without < need + kept + B * 256 * D * (n + 1) * 4 + 512


def test_where_the_walk_has_all_segments_in_one():
    """Enough channels and few tokens: no segments, so that the parts are all there is beside the sums."""
    B, L, D, N = 64, 1024, 1536, 128
    need, _ = backward_bytes(B, L, D, N)
    assert need <= GIB + 3 * B * D * 128 * 4 + 4096
    assert B * L * D * 128 * 128 * 8 // 1024 > 10 * need  # (what the parts of all tokens would be)
    # within the bound nothing is cut: all tokens' parts, and the sums
    B, L, D, N = 4, 1024, 1536, 16
    need, _ = backward_bytes(B, L, D, N)
    assert need >= B * L * D * 2


def test_no_tokens():
    assert backward_bytes(2, 0, 64, 16)[0] == 0
