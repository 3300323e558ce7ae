"""Which kernel prefix attention takes with several nodes a sequence, and how it splits the
prefixes (pz_prefixplan.h)."""
import pytest

from test_prefix_plan import FEW, SOME, WIDE, kernel, program  # noqa: F401 (fixtures)


def test_forms_of_the_gpu_cases(kernel):  # noqa: F811
    # test_gpu_prefix_wide.py: nodes of many sequences, of none that is seen, replayed
    for T in (3, 5):
        for D in (64, 128):
            assert kernel(4, 140, T, 32, 8, 224, D) == WIDE
    # drafts under prompts
    for D in (64, 128):
        assert kernel(4, 64, 5, 32, 8, 2128, D) == WIDE
    # own positions in splits
    for D in (64, 128):
        assert kernel(1, 128, 3, 32, 8, 2128, D) == WIDE
    # more rows than the workspace: 403 sequences, then 97
    assert kernel(3, 403, 5, 32, 8, 176, 128) == WIDE
    assert kernel(3, 97, 5, 32, 8, 176, 128) == SOME


def test_ranges_that_are_empty_count(kernel):  # noqa: F811
    """The host knows how many ranges there are, not how many hold a sequence."""
    assert kernel(1, 256, 1, 32, 8, 4096, 128) == WIDE
    assert kernel(150, 256, 1, 32, 8, 4096, 128) == FEW


def time_of(wgs, tiles, others, S, cu=256):
    """The rule's time of S splits, in tiles."""
    one = -(-tiles // S) + 6
    return max(-(-wgs * S // cu) * one, (wgs * S * one + others) // cu + 18)


@pytest.mark.parametrize("others", [0, 576, 4608, 100000])
@pytest.mark.parametrize("wgs", [1, 8, 32, 100, 128, 256, 300, 5000])
def test_no_other_splits_take_less_time(program, wgs, others):  # noqa: F811
    for tiles in (1, 8, 129, 513, 1025, 1 << 22):
        most = min(64, tiles // 8)
        S = program("splits", wgs, tiles, others, most)
        assert 1 <= S <= max(most, 1)
        got = time_of(wgs, tiles, others, S)
        for other in range(1, most + 1):
            t = time_of(wgs, tiles, others, other)
            assert got < t or got == t and S <= other, (tiles, S, other)


def test_whole_rounds(program):  # noqa: F811
    """Long prefixes and nothing beside them: the workgroups are a whole number of rounds."""
    for wgs in (4, 8, 32, 64, 128, 256, 512):
        S = program("splits", wgs, 1 << 20, 0, 64)
        assert wgs * S % 256 == 0, (wgs, S)
