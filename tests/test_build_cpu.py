"""When the library and the extension module are built."""
import os

import pytest

from rustorch_b200 import build as b


@pytest.fixture(scope="module", autouse=True)
def built():
    b.build()


def test_up_to_date_after_a_build():
    """Also where the newest file is the one with the compiler's flags: objects
    older than it are compiled again, and the next build finds nothing to do."""
    assert not b.needs_build() and not b.ops_stale()


def test_objects_are_as_new_as_the_flags():
    flags = os.path.getmtime(b.__file__)
    assert all(os.path.getmtime(b._obj(s)) >= flags for s in b._sources() if os.path.exists(b._obj(s)))
