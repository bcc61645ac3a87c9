"""Byte arrays in LDS are read and written as wider words through casts: each must state its alignment itself (a char array has that of one
byte, and where it lands then depends on what else the kernel declares)."""
import glob
import os
import re

from helpers import ROOT


def test_byte_arrays_in_lds_state_their_alignment():
    seen, bare = 0, []
    for path in sorted(glob.glob(os.path.join(ROOT, "image_caption_amd", "csrc", "*.h*"))):
        with open(path) as f:
            for n, line in enumerate(f, 1):
                m = re.search(r"__shared__\s+(.*?)\b(?:unsigned |signed )?char\s+\w+\[[^\]]", line)     # (arrays of the launch's own size, [], start LDS)
                if m:
                    seen += 1
                    if "aligned(16)" not in m.group(1):
                        bare.append(f"{os.path.basename(path)}:{n}")
    assert seen >= 2 and not bare, bare
