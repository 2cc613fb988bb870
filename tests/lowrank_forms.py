"""Which kernels a call of the shared projection runs, from the rules themselves (csrc/lowrank_rules.h, plain C++ that is compiled here), and
the sizes that together reach every one of them."""
import os
import subprocess

from conftest import PKG

TYPES = {'f32': 4, 'bf16': 6, 'f16': 7}

PROGRAM = r'''
#include "lowrank_rules.h"
#include <cstdio>
using namespace scs;
static void shrink(const scs_lowrank& p, int64_t K) {
    if (p.rows == 0) return;
    if (p.rows <= kDotRows) { printf("shrink dots,"); return; }
    const ShrinkForm f = shrink_form(p, K);
    printf("shrink jt%d mt%d w%d,", rank_tiles(p.rank), f.mt, f.waves);
}
static void project(const scs_lowrank& p, int64_t K, int64_t N, const char* way) {
    if (p.rows == 0) return;
    const Few f = few_of(p, K, N);
    if (f.mt) printf("few mt%d %s %s,", f.mt, f.splits > 1 ? "splits" : "one", way);
    else if (p.dtype == SCS_F32) printf("tiles32 %dx%d %s %s,", f32_rows(p.rows, N), f32_columns(N), N % 4 ? "odd" : "even", way);
    else printf("tiles %d %s %s,", tile16(p.rows, N), N % 8 ? "odd" : "even", way);
}
int main() {
    scs_lowrank p{};
    long long rows, in, out;
    int t, rank, adapters, requests;
    while (scanf("%d %lld %lld %lld %d %d %d", &t, &rows, &in, &out, &rank, &adapters, &requests) == 7) {
        p.dtype = t; p.rows = rows; p.in_features = in; p.out_features = p.ldw = out; p.rank = rank; p.n_adapters = adapters; p.n_requests = requests;
        shrink(p, in);
        project(p, in, out, "forward");
        shrink(p, out);
        const Few f = few_of(p, out, in);
        const int jt = rank_tiles(rank);
        if (rows && requests && few_beside_wgrad(p, f)) printf("few and gradients mt%d jt%d,", f.mt, jt);
        else if (rows && requests && tiles_beside_wgrad(p, f)) printf("tiles and gradients jt%d %s,", jt, in % 8 ? "odd" : "even");
        else {
            if (requests) project(p, out, in, "back");
            printf("gradients %s jt%d,", wgrad_block_rows(p) ? "blocks" : "direct", jt);
        }
        printf("\n");
    }
}
'''


def forms(calls, where):
    """A set of forms for each (type, rows, in, out, rank, adapters, requests), forward and backward with every gradient; operands at 16 bytes."""
    src, exe = os.path.join(str(where), 'forms.cpp'), os.path.join(str(where), 'forms')
    with open(src, 'w') as f:
        f.write(PROGRAM)
    subprocess.check_call(['g++', '-O1', '-std=c++17', '-Wno-unused-function', '-I', os.path.join(PKG, 'csrc'), src, '-o', exe])
    text = ''.join('%d %s\n' % (TYPES[c[0]], ' '.join(str(v) for v in c[1:])) for c in calls)
    out = subprocess.run([exe], input=text, capture_output=True, text=True, check=True).stdout
    return [set(line.strip(',').split(',')) for line in out.splitlines()]


def every_form(t):
    """All forms that a type's kernels are compiled in."""
    both = ('forward', 'back')
    want = {'shrink dots'}
    for jt in (1, 2, 4, 8):
        most = 16 if jt <= 2 else 8
        want |= {'shrink jt%d mt1 w%d' % (jt, w) for w in (4, 8, most)}
        if jt <= 2:
            want |= {'shrink jt%d mt2 w%d' % (jt, w) for w in (4, 8)}
        want |= {'gradients direct jt%d' % jt, 'gradients blocks jt%d' % jt}
    # (of one or two row tiles and up to two rank tiles backward: the launch that forms the gradients as well)
    want |= {'few mt%d %s %s' % (mt, s, way) for mt in ((1, 2) if t == 'f32' else (1, 2, 3, 4)) for s in ('one', 'splits') for way in both}
    want |= {'few and gradients mt%d jt%d' % (mt, jt) for mt in (1, 2) for jt in (1, 2)}
    if t == 'f32':
        want |= {'tiles32 %dx%d %s %s' % (mt, nt, e, way) for mt in (1, 2) for nt in (4, 5, 6, 7, 8) for e in ('even', 'odd') for way in both}
    else:
        want |= {'tiles %d %s %s' % (b, e, way) for b in (64, 128, 256) for e in ('even', 'odd') for way in both}
        want |= {'tiles and gradients jt%d %s' % (jt, e) for jt in (1, 2) for e in ('even', 'odd')}
    return want


# (rows, in, out, rank): beside the other sizes of test_gpu_lowrank.py these reach what a kernel is compiled for
SIZES = {
    'any': [(600, 1950, 72, 24), (600, 1000, 72, 40), (600, 1000, 72, 100), (16500, 1930, 64, 8), (16500, 1930, 61, 24), (16400, 64, 40, 8), (16400, 67, 35, 24)],
    # tiles of 64 and of 128 rows, every width, and its odd neighbour; few rows with much to multiply
    'f32': [(rows, n_in - odd, n_out - odd, rank) for rows in (12300, 32700) for odd in (0, 1)
            for n_in, n_out, rank in ((64, 112, 8), (112, 64, 24), (80, 96, 5), (96, 80, 40), (128, 128, 17))] +
           [(300, 1500, 1500, 8), (300, 1500, 1500, 24), (300, 1500, 1500, 40), (300, 16500, 130, 40), (300, 130, 16500, 40), (500, 2400, 72, 24)],
    '16 bits': [(10, 200, 300, 40), (20, 200, 300, 40), (20, 2056, 1500, 40), (60, 640, 2100, 8), (12, 100, 200, 24), (25, 100, 200, 24), (600, 64, 80, 24),
                (6200, 512, 520, 24), (6200, 515, 517, 8), (24700, 512, 264, 8), (24700, 517, 261, 24)],
}


def sizes(t):
    return SIZES['any'] + SIZES['f32' if t == 'f32' else '16 bits']


def requests(rows):
    """Offsets and adapters (of three) of five requests that end inside tiles; the last rows belong to none."""
    return [0, rows // 50 + 1, rows // 9 + 2, rows // 3 + 1, rows // 2 + 1, rows - rows // 40], [1, 2, 0, -1, 1]
