"""GPU suite: the control of the pages at the ends of its arguments' ranges."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_hip_pages import NONE_FREE, ints  # noqa: E402


@pytest.fixture(scope="module")
def H():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from jukebox_amd import _lib, hip_ops
    _lib.lib()          # fail loudly if the extension is missing
    return hip_ops


@pytest.mark.parametrize("page", [1_200_000_000, 2 ** 30, 2 ** 30 + 1, 2 ** 31 - 1])
def test_a_page_as_long_as_lengths_get(H, page):
    """A sequence that fills the only page and grows by five: a second page is asked for, and there is none -- nothing changes.  The length and
    the page together pass 2^32."""
    table, lens, ref, status = ints([[0, -1]]), ints([min(page, 0x7fff0000 - 5)]), ints([1]), ints([0])
    full = int(lens) == page
    slots = H.pages_extend(table, lens, ref, ints([0, 5]), page, 8, status)
    torch.cuda.synchronize()
    if full:
        assert int(status) == NONE_FREE and slots.tolist() == [-1] * 8 and table.tolist() == [[0, -1]] and ref.tolist() == [1] and int(lens) == page
    else:               # room behind the last token
        n = 0x7fff0000 - 5
        assert int(status) == 0 and slots.tolist() == [n, n + 1, n + 2, n + 3, n + 4, -1, -1, -1] and table.tolist() == [[0, -1]] and ref.tolist() == [1]
    # the first tokens of an empty one
    table, lens, ref, status = ints([[-1, -1]]), ints([0]), ints([0]), ints([0])
    slots = H.pages_extend(table, lens, ref, ints([0, 3]), page, 3, status)
    assert int(status) == 0 and slots.tolist() == [0, 1, 2] and table.tolist() == [[0, -1]] and ref.tolist() == [1] and lens.tolist() == [3]
