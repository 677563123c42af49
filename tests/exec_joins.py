"""Where a branch around masked lanes ends, read from a kernel's listing.

`s_cbranch_execz L` is taken with no lane enabled, and the block at L gives the lanes back with an `s_or_b64 exec, exec, ..` of its
own. A vector instruction in front of that does nothing for a wave that took the branch: the register allocator of this compiler has put
copies there (from ordinary to accumulation registers, next to saved scalar registers), and what the wave read back was not what it had
kept. `early_vector_work` finds such blocks."""
import re

# these work whatever the lanes
ANY_LANES = re.compile(r"v_(readlane|writelane|readfirstlane)_b32|s_")


def early_vector_work(listing):
    """[(label, instruction)] of vector instructions between a label that s_cbranch_execz goes to and the block's exec restore."""
    targets = set(re.findall(r"s_cbranch_execz\s+(\.LBB\w+)", listing))
    found = []
    for block in re.split(r"\n(?=\.LBB\w+:)", listing):
        label = block.split(":", 1)[0].strip()
        if label not in targets:
            continue
        early = []
        for line in block.split("\n")[1:]:
            line = line.split(";", 1)[0].strip()
            if not line or line.startswith("."):
                continue
            if re.match(r"s_(or|mov|xor|andn2|and)_b64 exec, |s_or_saveexec_b64 ", line):
                found += [(label, x) for x in early]
                break
            if re.match(r"s_(cbranch|branch|endpgm|setpc)", line):
                break
            if not ANY_LANES.match(line):
                early.append(line)
    return found
