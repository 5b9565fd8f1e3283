"""More of what the cache operators' Python entry points check, without a GPU (as test_cache_args)."""
import pytest

from test_cache_args import Recorder, attn_args, core, evict_args, sent  # noqa: F401


class Refusing(Recorder):
    """A library that answers 0 for a workspace, with or without a reason."""

    def __init__(self, why):
        super().__init__()
        self.why = why

    def dc_prefix_attention_ws(self, h, a):
        return 0

    def dc_last_error(self, h):
        return self.why


def test_workspace_of_refused_arguments_raises(core, P):  # noqa: F811
    a = attn_args()
    core.L = Refusing(b"prefix_attention: rows 17")
    with pytest.raises(P.DeviceError, match="rows 17"):
        core.prefix_attention_ws(**a)
    core.L = Refusing(b"")
    assert core.prefix_attention_ws(**a) == 0


@pytest.mark.parametrize("budget, recent, passed", [
    (2 ** 31 - 1, 0, (2 ** 31 - 1, 0)), (2 ** 31, 7, (2 ** 31 - 1, 7)), (2 ** 63, 2 ** 40, (2 ** 31 - 1, 2 ** 31 - 1)),
    (9, 2 ** 31, (9, 2 ** 31 - 1)), (-2 ** 40, 0, (-1, 0)), (9, -2 ** 33, (9, -1))])
def test_budgets_beyond_32_bits(core, P, budget, recent, passed):  # noqa: F811
    """No limit (a budget as large as can be) is a budget; what the library refuses stays what it refuses."""
    core.cache_evict_dev(**evict_args(n=9), budget=budget, recent=recent)
    assert sent(core, P, "dc_cache_evict_dev", "CACHE_EVICT")[-3:-1] == passed
