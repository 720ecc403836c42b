"""PagedTransformer.generate when it cannot finish."""
import pytest

from test_gpu_paged_decode import _model

pytestmark = pytest.mark.gpu


def test_generate_that_fails_leaves_no_sequence(cuda_device):
    """A sequence that generate opened itself is nobody's if it raises: its slot and pages are free again."""
    from mira_b200.paged import OutOfPages
    w, model = _model("f32", max_pages=2)
    pages = model.cache.pages
    for prompt, new, error in (([1, 2, 50], 1, ValueError), ([0] * 17, 1, OutOfPages), ([3, 4], 20, OutOfPages), ([], 1, ValueError)):
        with pytest.raises(error):
            model.generate(prompt, new)
        assert not pages.live.any() and pages.used_pages() == 0
    # a sequence that was there keeps what it has
    slot, out = model.generate([5, 6], 3)
    with pytest.raises(OutOfPages):
        model.generate(out[-1:], 20, slot=slot)
    assert pages.live[slot] and pages.lengths[slot] == 16
    other, again = model.generate([5, 6], 3)
    assert other != slot and again == out
    model.close()
