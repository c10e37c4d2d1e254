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


def test_rows_are_staged_behind_all_queries_of_their_half():
    """Outputs are laid where queries were.  The last product has waited for all of a half's queries; a block without a key tile has
    no product, and waits for the queries themselves."""
    text = _source("kv4_attention_tc5.cu")
    staged = text.index("unsigned char* stage = Qs")
    before = text[text.rindex("pdl_launch_dependents()", 0, staged):staged]
    assert re.search(r"if \(n_tiles > 0\) \{[^}]*mbar_wait\(&o_done\[h\][^}]*\} else \{[^}]*mbar_wait\(&q_full\[h\]", before)
