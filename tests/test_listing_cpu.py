"""What the compiler makes of kernels whose results or safety hang on it, read from listings of the library's own code (no GPU needed)."""
import collections
import os
import re
import shutil
import subprocess

import pytest

from hortimapping_amd import build as hb

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
pytestmark = pytest.mark.skipif(shutil.which(HIPCC) is None, reason="no hipcc")


def kernel(listing, name):
    """Body of the one kernel whose mangled name holds `name`."""
    starts = [m for m in re.finditer(r"^(_Z\S+):", listing, re.M) if name in m[1]]
    assert len(starts) == 1, [m[1] for m in starts]
    body = listing[starts[0].end():]
    return body[:body.index(".Lfunc_end")]


def test_transformed_points_do_not_hang_on_the_compilers_choice(tmp_path):
    """The sums of products of both point transforms round the same way whether the compiler may fuse products into sums across
    statements (its default here), within one, or not at all: all fusing is written out."""
    modes = ("fast-honor-pragmas", "on", "off")
    count = {}
    for contract in modes:
        out = str(tmp_path / f"{contract}.s")
        subprocess.run([HIPCC] + hb.FLAGS + [f"-ffp-contract={contract}", "-S", "--cuda-device-only", os.path.join(hb.CSRC, "hm_render.hip"),
                                             "-o", out], check=True, capture_output=True)
        listing = open(out).read()
        for name in ("k_transform_points", "k_sample_rays"):
            count[name, contract] = collections.Counter(re.findall(r"^\s+(v_(?:fma|mul|add|sub)\w*_f32)", kernel(listing, name), re.M))
    for name in ("k_transform_points", "k_sample_rays"):
        assert count[name, modes[0]] == count[name, "on"] == count[name, "off"] and sum(count[name, "off"].values()) >= 13
