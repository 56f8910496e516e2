"""Register spills of the sequence operators' kernels, read from the object files of the in-tree build as in
tests/test_kernel_resources.py: the forms that are known to spill, with how many registers at most, and none beside them."""
import re
import subprocess

import pytest

from test_kernel_resources import built, pytestmark  # noqa: F401

# <rows, wavefronts, halves, backwards, whole vectors> of float32, <rows, backwards, whole vectors> of float64
ATTENTION = {
    r"sums_f32<96, 8, 1, \w+, true>": 8,
    r"chunks_f32<(32, [48]|64, 8), 1, \w+, false>": 24, r"chunks_f32<(96|128), 8, [12], \w+, false>": 52, r"sums_f32<(96|128), 8, 1, \w+, false>": 8,
    r"chunks_f64<(192|256), \w+, true>": 128, r"chunks_f64<64, \w+, false>": 56, r"chunks_f64<192, \w+, false>": 168, r"chunks_f64<256, \w+, false>": 272,
    r"sums_f64<256, \w+, false>": 64,
}
NORM = {r"image_backward<double, \d+, [12], \d+, [012]>": 4, r"team_backward<double, 2, 8, true, [012], \w+>": 64}


def names(kernels):
    """The kernels' names with their template arguments, as c++filt writes them."""
    text = subprocess.run(["c++filt"], input="\n".join(k[0] for k in kernels), capture_output=True, text=True, check=True).stdout
    return [re.sub(r"^.*?(\w+<[^>]*>|\w+)\(.*$", r"\1", n.replace("(bool)1", "true").replace("(bool)0", "false").replace("(int)", "")) for n in text.splitlines()]


@pytest.mark.parametrize("unit,known", [("rotary", {}), ("decay_attention", ATTENTION), ("group_norm", NORM)])
def test_only_the_known_forms_spill(built, unit, known):  # noqa: F811
    assert built[unit], unit
    bad = []
    for name, (_, _, spilled, scratch) in zip(names(built[unit]), built[unit]):
        if not spilled and not scratch:
            continue
        rule = next((r for r in known if re.fullmatch(r, name)), None)
        if rule is None or spilled > known[rule]:
            bad.append((name, spilled, scratch))
    assert not bad, bad
