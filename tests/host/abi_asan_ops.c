/* Host side of the tensor operators (ivae_linear, ivae_layer_norm, ivae_dropout) under AddressSanitizer + UBSan: size queries over a random
 * walk of shapes (valid, degenerate, huge), NULL arguments, and -- only when no device is visible -- whole calls with fake device
 * pointers, which must come back as IVAE_E_HIP after every choice of tiles, splits and workspace pieces has been made on the host.
 * Prints "abi_asan_ops: OK" and exits 0 when every check held. */
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#include "../../include/ivae_amd.h"

int hipGetDeviceCount(int* n);

static int fails = 0;
#define CHECK(c, ...) do { if (!(c)) { ++fails; fprintf(stderr, "abi_asan_ops: " __VA_ARGS__); fputc('\n', stderr); } } while (0)

static uint64_t rng = 0x2545F4914F6CDD1Dull;
static uint32_t rnd(void) { rng ^= rng << 13; rng ^= rng >> 7; rng ^= rng << 17; return (uint32_t)(rng >> 11); }
static int64_t pick(const int64_t* v, int n) { return v[rnd() % n]; }

int main(void) {
    int devices = 0;
    if (hipGetDeviceCount(&devices) != 0) devices = 0;
    const int64_t rows[] = {-1, 0, 1, 2, 16, 17, 63, 64, 65, 127, 128, 256, 1000, 1531, 4096, 8192, 65536, 1 << 20, (int64_t)1 << 29, ((int64_t)1 << 29) - 1,
                            (int64_t)1 << 31, (int64_t)1 << 40, ((int64_t)1 << 40) + 1};
    const int64_t width[] = {-3, 0, 1, 7, 8, 16, 50, 63, 64, 65, 200, 256, 777, 1001, 1024, 4096, 4100, 16384, 16385, 1 << 20, (1 << 21) + 8, 1 << 24, (1 << 24) + 1};
    char* fake = (char*)(uintptr_t)0x100000000ull;      /* never dereferenced on the host */
    for (int it = 0; it < 60000; ++it) {
        IvaeLinear l;
        memset(&l, 0, sizeof l);
        l.rows = pick(rows, 23);
        l.in_features = (int32_t)pick(width, 23);
        l.out_features = (int32_t)pick(width, 23);
        l.dtype = (int)(rnd() % 5) - 1;
        l.activation = (int)(rnd() % 8) - 1;
        l.slope = .1f;
        l.ldx = rnd() % 8 == 0 ? pick(width, 23) : l.in_features;
        l.ld_residual = rnd() % 8 == 0 ? pick(width, 23) : l.out_features;
        l.lddy = rnd() % 8 == 0 ? pick(width, 23) : l.out_features;
        size_t f = 0, b = 0;
        const int rf = ivae_linear_workspace_bytes(&l, 0, &f), rb = ivae_linear_workspace_bytes(&l, 1, &b);
        CHECK(rf == rb && rf <= 0 && rf >= IVAE_E_BADTYPE, "ivae_linear_workspace_bytes -> %d / %d", rf, rb);
        if (rf == 0) CHECK(f < ((size_t)1 << 60) && b < ((size_t)1 << 60), "workspace of %zu / %zu bytes", f, b);
        if (devices == 0 && (rf != 0 || l.rows <= 8192)) {
            const int y = ivae_linear(&l, fake, fake, fake, it & 1 ? fake : NULL, fake, it & 2 ? fake : NULL, fake, f, NULL);
            const int g = ivae_linear_backward(&l, fake, fake, fake, fake, it & 4 ? fake : NULL, it & 8 ? fake : NULL, it & 16 ? fake : NULL, fake, b, NULL);
            CHECK(rf ? y == rf && g == rf : (y == IVAE_OK || y == IVAE_E_HIP) && (g == IVAE_OK || g == IVAE_E_HIP), "ivae_linear -> %d, backward -> %d, sizes -> %d", y, g, rf);
            if (rf == 0 && f > 0) CHECK(ivae_linear(&l, fake, fake, NULL, NULL, fake, NULL, fake, f - 1, NULL) == (l.rows ? IVAE_E_WORKSPACE : IVAE_OK), "small workspace");
            if (rf == 0 && b > 0) CHECK(ivae_linear_backward(&l, fake, fake, fake, fake, fake, fake, fake, fake, b - 1, NULL) == IVAE_E_WORKSPACE, "small workspace, backward");
        }
        IvaeNorm n;
        memset(&n, 0, sizeof n);
        n.rows = pick(rows, 23);
        n.width = (int32_t)pick(width, 23);
        n.dtype = (int)(rnd() % 5) - 1;
        n.weight_f32 = rnd() & 1;
        n.eps = 1e-5f;
        n.ldx = n.lddy = n.ld_residual = n.width;
        size_t w = 0;
        const int rn = ivae_layer_norm_workspace_bytes(&n, &w);
        CHECK(rn <= 0 && rn >= IVAE_E_BADTYPE, "ivae_layer_norm_workspace_bytes -> %d", rn);
        if (devices == 0) {
            const int y = ivae_layer_norm(&n, fake, fake, fake, fake, (float*)fake, NULL);
            const int g = ivae_layer_norm_backward(&n, fake, fake, (float*)fake, fake, NULL, fake, it & 1 ? fake : NULL, it & 2 ? fake : NULL, fake, w, NULL);
            CHECK(rn ? y == rn && g == rn : (y == IVAE_OK || y == IVAE_E_HIP) && (g == IVAE_OK || g == IVAE_E_HIP), "ivae_layer_norm -> %d, backward -> %d, sizes -> %d", y, g, rn);
            const int d = ivae_dropout((int)(rnd() % 5) - 1, pick(rows, 23), fake, NULL, fake, (double)(rnd() % 12) / 10. - .1, rng, rng, NULL, NULL);
            CHECK(d <= 0 && d >= IVAE_E_BADTYPE, "ivae_dropout -> %d", d);
        }
    }
    size_t o;
    CHECK(ivae_linear_workspace_bytes(NULL, 0, &o) < 0 && ivae_layer_norm_workspace_bytes(NULL, &o) < 0, "NULL size queries");
    CHECK(ivae_linear(NULL, NULL, NULL, NULL, NULL, NULL, NULL, NULL, 0, NULL) < 0 && ivae_linear_backward(NULL, NULL, NULL, NULL, NULL, NULL, NULL, NULL, NULL, 0, NULL) < 0 &&
          ivae_layer_norm(NULL, NULL, NULL, NULL, NULL, NULL, NULL) < 0 && ivae_dropout(0, 4, NULL, NULL, NULL, .1, 0, 0, NULL, NULL) < 0, "NULL calls");
    if (fails) return 1;
    printf("abi_asan_ops: OK (%s)\n", devices ? "a device is visible: size queries only" : "whole host paths");
    return 0;
}
