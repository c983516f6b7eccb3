// Reads pairs of tensors of rows (address, element size, heads, rows, strides of a head and of a row, 128 elements a head), prints 1 where pg_rows_meet says that they meet
#include <stdio.h>

#include "../../spy_amd/csrc/rows_meet.h"

int main() {
    spy_hip_tensor t[2] = {};
    for (;;) {
        for (int i = 0; i < 2; i++) {
            long long at, es, nh, nr, h, r;
            if (scanf("%lld %lld %lld %lld %lld %lld", &at, &es, &nh, &nr, &h, &r) != 6) return 0;
            t[i].data = (void *)at;
            t[i].ne[0] = 128; t[i].ne[1] = nh; t[i].ne[2] = nr; t[i].ne[3] = 1;
            t[i].nb[0] = es; t[i].nb[1] = h; t[i].nb[2] = r; t[i].nb[3] = r * nr;
        }
        printf("%d\n", pg_rows_meet(&t[0], &t[1]) ? 1 : 0);
    }
}
