// prints how many portions in_portions makes of a total, and what they add up to; gives up after 1000 (so would a caller that queues launches for ever)
#include <stdio.h>

#include "portions.h"

int main() {
    unsigned long long total;
    unsigned most, stop;
    while (scanf("%llu %u %u", &total, &most, &stop) == 3) {
        unsigned long long calls = 0, sum = 0, next = 0;
        const int r = nb::in_portions(total, most, [&](uint32_t at, uint32_t n) {
            if (at != next || !n || n > most || ++calls > 1000) return 1;
            sum += n; next += n;
            return calls == stop ? 7 : 0;
        });
        printf("%d %llu %llu\n", r, calls, sum);
    }
    return 0;
}
