"""What autograd has to know of the paged kernels."""
import pytest

import test_paged_autograd_cpu as on

pytestmark = pytest.mark.gpu


def test_out_is_known_to_autograd():
    on.out_is_known_to_autograd("cuda")
