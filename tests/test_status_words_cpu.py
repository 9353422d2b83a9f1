"""Every kernel file with bounded waits reports to the host's word and is asked for its own."""
import re

from holon_b200.kernels import cuda
from holon_b200.kernels.build import CSRC


def test_every_file_with_bounded_waits_is_asked():
    defined = {}
    for path in sorted(CSRC.glob("*.cu")):
        for name in re.findall(r"HB_DEFINE_STATUS_MIRROR\((\w+)_status_mirror\)", path.read_text()):
            defined[name] = path
    assert {"hb_attention_tcgen05", "hb_attention_rows", "hb_attention_prefix"} <= set(defined)
    handed = (CSRC / "status.cu").read_text()
    python = open(cuda.__file__).read()
    for name, path in defined.items():
        assert f"{name}_status_mirror(device)" in handed, f"{path.name} is not handed the host's word"
        assert f'"{name}_status"' in python and f"int {name}_status(unsigned int*" in path.read_text(), f"{path.name} is not asked for its word"
