"""Which kernel glm53f_fwd_gemm_bf16_fused launches, restated: the tests choose sizes by it that reach every kernel, and hold
the kernels that the library is built with to the ones that sizes reach.

A kernel of the weight-streaming kind is ("stream", CK, NT, T, KS, ANY), of tiles ("tile", BM, BN, BK, FAST, TAIL)."""
import itertools
import re

CUS = 256
SHAPES = [(64, 32, 0.20, 0.33), (64, 64, 0.29, 0.43), (128, 64, 0.39, 0.67), (128, 128, 0.56, 0.85), (128, 256, 0.96, 1.31),
          (256, 256, 1.85, None)]
BK = {True: (128, 128, 128, 64, 64, 32), False: (128, 128, 64, 64, 64)}


def ceil(a, b):
    return -(-a // b)


def _stream(rows, n, k, groups, any_):
    tiles, nt = ceil(n, 16) * groups, 1 if rows <= 16 else 2 if rows <= 32 else 4
    tmax = 8 if nt == 1 else 4

    def split(ck, ks, tmax):
        for t in (8, 4, 2):
            if tmax >= t and tiles > t // 2 * CUS:
                return "stream", ck, nt, t, ks, any_
        return "stream", ck, nt, 1, ks, any_

    if tiles <= CUS and (k >= 1024 if any_ else k % 1024 == 0):
        row_tiles = nt if rows <= 64 else ceil(rows, 16)
        if not any_ and k % 2048 == 0 and (nt == 1 or tiles * row_tiles <= CUS):
            return "stream", 256, 1, 1, 8, any_
        return "stream", 128, nt, 1, 8, any_
    if k >= 512 if any_ else k % 512 == 0:
        return split(256, 4, 8) if not any_ and k % 1024 == 0 else split(128, 4, tmax)
    return split(128, 1, tmax)


def kernel_of(rows, n, k, groups=1, aligned=True):
    """aligned: x and w at 16-byte addresses with strides that are multiples of 8."""
    if k < 8:
        return ("short",)
    if rows <= 64 or (rows <= 256 and ceil(n, 16) * ceil(rows, 64) * groups <= CUS and k >= 512):
        whole = k < 512 or k % (1024 if ceil(n, 16) * groups <= CUS and k >= 1024 else 512) == 0
        return _stream(rows, n, k, groups, not (aligned and n % 16 == 0 and k % 128 == 0 and whole))
    fast = aligned and k % 8 == 0
    times = [ceil(ceil(rows, bm) * ceil(n, bn) * groups, CUS) * (a if fast else b) for bm, bn, a, b in SHAPES[:6 if fast else 5]]
    i = times.index(min(times))
    return "tile", *SHAPES[i][:2], BK[fast][i], fast, fast and k % (128 if i <= 2 else 64) != 0


def built(path):
    """The kernels of the fused product in the library, by the names of their descriptors."""
    data = open(path, "rb").read()
    found = set()
    for m in re.finditer(rb"stream_kernelILi(\d+)ELi(\d+)ELi(\d+)ELi(\d+)ELb([01])EN9fwd_fused[^\0]*?\.kd\0", data):
        found.add(("stream", *map(int, m.groups()[:4]), m[5] == b"1"))
    for m in re.finditer(rb"fwd_fused[^\0]*?tile_kernelILi(\d+)ELi(\d+)ELi\d+ELi\d+ELi\d+ELi(\d+)ELi\d+ELb([01])ELb([01])E[^\0]*?\.kd\0", data):
        found.add(("tile", *map(int, m.groups()[:3]), m[4] == b"1", m[5] == b"1"))
    return found


def sizes():
    rows = [1, 16, 17, 32, 33, 64, 65, 100, 128, 200, 256, 257, 384, 512, 700, 1024, 1500, 2048, 3000, 4096, 8192]
    ns = [16, 160, 1024, 2048, 2500, 4096, 4112, 6000, 8192, 8208, 16384, 16400, 24640, 65536]
    ks = [8, 128, 384, 512, 520, 576, 1001, 1024, 1152, 1536, 2048, 4096, 8200]
    return itertools.product(rows, ns, ks, (True, False))


def reached():
    return {kernel_of(r, n, k, 1, a) for r, n, k, a in sizes()}


def cheapest():
    """Every kernel with the sizes of the least work that reach it, {kernel: (rows, n, k, aligned)}: tiles with several steps
    of k, of rows at any address an odd k."""
    found = {}
    for r, n, k, a in sorted(sizes(), key=lambda s: (s[0] + 64) * s[1] * s[2]):
        kernel = kernel_of(r, n, k, 1, a)
        if kernel[0] == "stream" or (k > 512 if a else k % 2):
            found.setdefault(kernel, (r, n, k, a))
    return found
