"""More of what the cache operators' Python entry points check, without a GPU (as test_cache_args)."""
import pytest

from test_cache_args import Recorder, attn_args, core  # noqa: F401


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
