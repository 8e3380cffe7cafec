"""Which form of the 4-bit product a call takes, without a GPU: the sizes of the GPU tests reach every one."""
import subprocess
from pathlib import Path

from tests import mx4_forms

CSRC = Path(__file__).resolve().parents[1] / "cleffa_amd" / "csrc"


def _forms(sizes, tmp_path):
    """(form with X in 4 bits, with X in bf16) of each (T, N), and all forms there are."""
    (tmp_path / "f.cpp").write_text('#include <cstdio>\n#include "mx4_forms.h"\nusing namespace clef_hip::mx4;\nint main() {\n'
                                    + "".join(f'puts(kForms4[form4({T}, {N})]); puts(kForms16[form16({T}, {N})]);\n' for T, N in sizes)
                                    + 'for (auto f : kForms4) puts(f);\nfor (auto f : kForms16) puts(f);\n}\n')
    subprocess.run(["g++", "-std=c++17", "-I", str(CSRC), str(tmp_path / "f.cpp"), "-o", str(tmp_path / "f")], check=True)
    out = subprocess.run([str(tmp_path / "f")], check=True, capture_output=True, text=True).stdout.splitlines()
    n = 2 * len(sizes)
    return list(zip(out[:n:2], out[1:n:2])), out[n:n + 9], out[n + 9:]


def test_every_form_has_a_size(tmp_path):
    got, all4, all16 = _forms([*mx4_forms.X4.values(), *mx4_forms.X16.values()], tmp_path)
    n = len(mx4_forms.X4)
    assert [g[0] for g in got[:n]] == list(mx4_forms.X4) and [g[1] for g in got[n:]] == list(mx4_forms.X16)
    assert sorted(mx4_forms.X4) == sorted(all4) and sorted(mx4_forms.X16) == sorted(all16)


def test_forms_of_a_layer(tmp_path):
    """One token, a batch, a request, a micro-batch against the widths of a layer."""
    sizes = {(1, 5120): ("rows 1x2", "rows 1x2 few"), (1, 14336): ("rows 2x4", "rows 1x4 few"), (45, 14336): ("rows 4x4", "rows 2x4/4"), (61, 5120): ("rows 2x4", "rows 2x4"),
             (256, 5120): ("tile 64x128", "tile 64x256"), (425, 10240): ("tile 256x128", "tile 128x256"), (1160, 5120): ("tile 256x128", "tile 128x256"),
             (1300, 10240): ("tile 256x256", "tile 128x256"), (4096, 14336): ("tile 256x128", "tile 128x256"), (2048, 14336): ("tile 256x256", "tile 64x256"), (1, 1): ("rows 1x1", "rows 1x1 few"),
             (1 << 20, 1): ("tile 256x128", "tile 128x256")}
    assert dict(zip(sizes, _forms(list(sizes), tmp_path)[0])) == sizes
