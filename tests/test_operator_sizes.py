"""Sizes that the library is asked for before any device work, over what the header allows."""
import subprocess
import sys

import pytest

from tests.conftest import PKG


@pytest.mark.parametrize("mxfp8", [0, 1])
def test_the_work_area_of_an_empty_decoding_step(mxfp8):
    """0 to 511 tokens are allowed, so a binding may ask for the size of an empty step's work area; in a process of its own, since
    a fault of the library would end this one."""
    code = (f"import sys; sys.path.insert(0, {PKG!r})\n"
            "from mok import _C\n"
            f"print(*(_C.lib.mokb_few_tokens_workspace_bytes(t, 256, 128, 2, {mxfp8}) for t in (0, 1, 16, 511, 512)))\n")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, (r.returncode, r.stderr)
    none, one, sixteen, most, too_many = map(int, r.stdout.split())
    assert 0 < none <= one <= sixteen < most and too_many == 0
