"""What the compiler made of kernels whose speed hangs on it: read from the built library's own metadata (no GPU needed)."""
import os
import re
import subprocess

import pytest

from marl_amd import _hip

READELF = '/opt/rocm/llvm/bin/llvm-readelf'


def _kernels(tmp_path):
    """{kernel: {key: number}} of every device image in the library."""
    data, out = open(_hip._LIB_PATH, 'rb').read(), {}
    starts = [m.start() for m in re.finditer(b'\x7fELF', data)][1:]          # the first is the library itself
    for a, b in zip(starts, starts[1:] + [len(data)]):
        image = tmp_path / 'image'
        image.write_bytes(data[a:b])
        text = subprocess.run([READELF, '--notes', str(image)], capture_output=True, text=True).stdout
        for block in text.split('- .agpr_count:')[1:]:
            name = re.search(r'\.name:\s+(\S+)', block)
            if name:
                out[name.group(1)] = {k: int(v) for k, v in re.findall(r'\.(\w+):\s+(\d+)\n', block)}
    return out


@pytest.mark.skipif(not os.path.exists(READELF), reason='no llvm-readelf')
def test_the_vector_actor_does_not_spill_its_weights(tmp_path):
    """Its scalar weight loads pulled to the top of the loop cost 540 spills, and five sixths of its speed."""
    found = {k: v for k, v in _kernels(tmp_path).items() if 'actor_forward_kernel' in k}
    assert len(found) == 2
    for name, v in found.items():
        assert v['sgpr_spill_count'] < 64 and v['vgpr_spill_count'] == 0 and v['private_segment_fixed_size'] == 0, (name, v)
