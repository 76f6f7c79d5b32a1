"""Without a GPU: what the serving step's calls (kernels.serving) make of arguments off the usual ones, and what they refuse,
through the Python functions, the C ABI and the METH_FASTCALL binding."""
import re
from pathlib import Path

import pytest
import torch

from kernels import _native, serving


@pytest.fixture(scope="module")
def lib():
    if not _native.library_path().exists():
        pytest.fail(f"{_native.library_path()} is not built: run `python slm-turbo_amd/build_lib.py`")
    return _native.load()


# =============================================================================
#  prompt attention
# =============================================================================
def test_rows_that_the_attention_cannot_read_are_copied():
    """Also those that torch calls contiguous: an odd address, an odd stride of a dim of one element."""
    flat = torch.arange(9000, dtype=torch.float32).half()
    for t in (flat[1:1 + 20 * 3 * 64].view(20, 3, 64), flat.as_strided((1, 3, 64), (195, 64, 1)), flat.as_strided((20, 1, 64), (64, 67, 1)),
              flat.as_strided((1, 1, 80), (3, 5, 1)), flat.as_strided((5, 2, 64), (128, 64, 1), 4), flat.as_strided((1, 2, 64), (1 << 29, 64, 1)),
              flat.as_strided((5, 2, 64), (130, 65, 1)), flat.as_strided((5, 2, 64), (128, 1, 2))):
        got = serving._rows16(t)
        assert torch.equal(got, t) and got.data_ptr() % 16 == 0
        assert got.stride() == (t.shape[1] * t.shape[2], t.shape[2], 1)
    for t in (flat[8:8 + 20 * 2 * 64].view(20, 2, 64), flat.as_strided((5, 2, 64), (256, 64, 1)), flat.as_strided((2, 5, 64), (64, 128, 1))):
        assert serving._rows16(t) is t


# =============================================================================
#  the sources
# =============================================================================
def test_inline_assembly_names_what_it_changes():
    """Every asm statement that writes m0 lists it (and memory, where it loads to LDS): the compiler may hold a value there."""
    csrc, seen = Path(serving.__file__).resolve().parents[1] / "csrc", 0
    for path in sorted([*csrc.glob("*.hip"), *csrc.glob("*.h")]):
        for statement in re.findall(r"\basm\b[^;]*?;", path.read_text()):
            if re.search(r"\bs_mov_b32 m0\b", statement):
                seen += 1
                outputs = statement.rsplit(":", 1)[1]
                assert '"m0"' in outputs and '"memory"' in outputs, f"{path.name}: {statement}"
    assert seen >= 4
