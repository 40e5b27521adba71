"""What autograd has to know of the paged kernels."""
import pytest

import test_paged_autograd_cpu as on

pytestmark = pytest.mark.gpu


def test_out_is_known_to_autograd():
    on.out_is_known_to_autograd("cuda")


def test_forward_mode_is_refused():
    on.forward_mode_is_refused("cuda")
