"""Results that lie over what the kernels read."""
import pytest

import test_paged_overlap_cpu as on

pytestmark = pytest.mark.gpu


def test_out_lies_anywhere():
    on.out_lies_anywhere("cuda")


def test_out_over_itself_is_refused():
    on.out_over_itself_is_refused("cuda")


def test_append_to_pages_over_themselves_is_refused():
    on.append_to_pages_over_themselves_is_refused("cuda")
