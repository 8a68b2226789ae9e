"""Host-side checks of the windowed operators' edge cases: the shared window arithmetic compiled as plain C."""
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent


def run_c(tmp_path, body):
    src = tmp_path / "walk.c"
    src.write_text('#include <stdio.h>\n#include <stdlib.h>\n#include "h3b_window.h"\n'
                   "static int sees(int j, int p, h3b_win w, int n) {\n"
                   "    int b = p - p % w.block;\n"
                   "    return j < n && j <= b + w.block - 1 + w.right && (j >= b - w.left || j < w.sinks);\n"
                   "}\n" + body)
    subprocess.run(["gcc", "-O1", "-I" + str(ROOT / "h3c_b200" / "csrc"), str(src), "-o", str(tmp_path / "walk")], check=True)
    done = subprocess.run([str(tmp_path / "walk")], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout


def test_a_block_is_looked_up_only_if_some_row_sees_some_key_of_it(tmp_path):
    """h3b_win_any against the definition, for every block of 64 keys of the tiles of 128 that a group of rows visits."""
    run_c(tmp_path, r"""
int main(void) {
    srand(1);
    for (int round = 0; round < 20000; round++) {
        int n = 1 + rand() % 900, rows = 1 + rand() % 200, p0 = n - rows;          /* the last rows of a sequence, as in the cache */
        h3b_win w = {rand() % 3 ? rand() % 300 : H3B_WIN_MAX, rand() % 3 ? 0 : rand() % 2 ? rand() % 100 : H3B_WIN_MAX,
                     rand() % 2 ? 0 : rand() % 300, rand() % 2 ? 1 : 1 + rand() % 150};
        h3b_win_row a = h3b_win_of(w, p0, n), z = h3b_win_of(w, n - 1, n);
        h3b_win_tiles t = h3b_win_tiles_of(w, p0, n - 1, n, 128);
        for (int i = 0; i < t.count; i++)
            for (int half = 0; half < 2; half++) {
                int k0 = h3b_win_tile(t, i) * 128 + half * 64, want = 0;
                for (int p = p0 < 0 ? 0 : p0; p < n && !want; p++)
                    for (int j = k0; j < k0 + 64 && !want; j++) want = sees(j, p, w, n);
                if (!h3b_win_any(z.hi, a.lo, z.s, k0, 64) != !want) {
                    printf("n %d rows %d window %d %d %d %d block %d: want %d", n, rows, w.left, w.right, w.sinks, w.block, k0, want);
                    return 1;
                }
            }
    }
    return 0;
}
""")
