"""Rules of the 4-bit cache's sources that no run can show to be kept."""
import os
import re

KERNELS = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "paged_batch_engine_b200", "csrc", "kernels")


def _source(name):
    with open(os.path.join(KERNELS, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def test_numbers_of_a_record_are_read_behind_a_barrier_of_the_warp():
    """A converting warp's lanes read numbers that other lanes of it stored: between the last store and the first read all
    lanes meet, and between the last read and the next record's first store."""
    text = _source("kv4_attention_tc5.cu")
    loop = text[text.index("for (int n = own; n < records; n += CONV)"):text.index("mbar_arrive(&full[st])")]
    stores = [m.end() for m in re.finditer(r"\bdst\[[^\]]*\]\s*=", loop)]
    reads = [m.start() for m in re.finditer(r"words<[^;]*\b(?:kn|vn)\b", loop)]
    assert len(stores) == 3 and len(reads) == 4                     # the code was found and understood
    assert max(stores) < min(reads) and "__syncwarp()" in loop[max(stores):min(reads)]
    assert "__syncwarp()" in loop[:min(stores)] and "__syncwarp()" in loop[max(reads):]
