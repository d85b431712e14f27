"""The cut of few long rows over workgroups (neural-motifs_amd/csrc/label_cut.h), compiled for the host with overflow checks."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r'''
#include <cstdio>
#include <initializer_list>
#include "label_cut.h"
int main()
{
    for (int rows = -1; rows <= 130; ++rows)
        for (long long base : {1ll, 16384ll, 20000ll, 65536ll, 100003ll, 1ll << 20, 1ll << 30, (1ll << 31) - 1})
            for (int off = -300; off <= 300; ++off) {
                const long long classes = base + off;
                if (classes < 1 || classes >= 1ll << 31) continue;
                const mh::ld::RowCut c = mh::ld::row_cut(rows, (int)classes);
                const bool cut = rows >= 1 && rows <= 128 && classes >= 16384;
                const bool fine = !cut ? c.nseg == 0
                                       : c.nseg >= 2 && c.nseg * rows <= 256 && c.length % 8 == 0 && (long long)c.nseg * c.length >= classes &&
                                             (c.nseg - 1ll) * c.length < classes;
                if (!fine) {
                    std::printf("rows %d classes %lld: %d of %d\n", rows, classes, c.nseg, c.length);
                    return 1;
                }
            }
    std::puts("fine");
    return 0;
}
'''


def test_every_class_is_in_one_part(tmp_path):
    (tmp_path / 'cut.cpp').write_text(PROGRAM)
    subprocess.check_call(['g++', '-std=c++17', '-O1', '-fsanitize=undefined', '-fno-sanitize-recover=all', '-I', os.path.join(ROOT, 'neural-motifs_amd', 'csrc'),
                           '-o', str(tmp_path / 'cut'), str(tmp_path / 'cut.cpp')])
    r = subprocess.run([str(tmp_path / 'cut')], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert r.returncode == 0 and 'fine' in r.stdout, r.stdout
