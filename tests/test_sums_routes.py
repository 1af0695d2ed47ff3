"""Which kernel, tiles and pieces a product takes whose fp32 sums are the result, from sizes alone (no GPU needed): what its route says where that leaves such sums, and every CU busy
where the tiles had to grow."""
from test_product_routes import run

WALK = '''
import itertools
WITH_SUMS = {(64, 96), (64, 128), (96, 96), (128, 128), (128, 192), (192, 128), (128, 256)}
rows = (1, 16, 33, 64, 100, 200, 333, 500, 777, 1024, 2048, 4096, 9000)
seen = set()
for m, n, k in itertools.product(rows, (64, 256, 576, 1024, 2048, 4096, 11008), (64, 576, 1728, 2048, 8192, 16384)):
    a, b = operand(m, k), operand(k, n)
    route, sums = host.product_route(a, b, "NN"), host.sums_route(a, b)
    kind, tile, *rest = sums.split()
    tile_m, tile_n = map(int, tile.split("x"))
    parts = int(rest[1]) if rest else 1
    assert kind == "large" or (tile_m, tile_n) in WITH_SUMS, (m, n, k, sums)
    tiles = -(-m // tile_m) * -(-n // tile_n)
    first, second = (route.split() + [""])[:2]
    if first == "large" or (first == "mid" and tuple(map(int, second.split("x"))) in WITH_SUMS):
        assert sums == route, (m, n, k, route, sums)
        seen.add(second)
    else:
        # as many pieces as there are CUs to take them and 512 of contraction for each, 8 at most
        assert parts == max(1, min(256 // tiles, k // 512, 8)), (m, n, k, route, sums)
        seen.add("grown")
    assert parts * 64 <= max(k, 64)
assert {"64x96", "96x96", "64x128", "grown"} <= seen, seen
'''


def test_the_routes_tiles_are_kept_and_grown_ones_go_in_pieces():
    run(WALK)


def test_what_no_kernel_takes():
    run('''
assert host.sums_route(operand(4, 64), operand(64, 36)) == "none"        # rows of the result that are no multiple of 8
assert host.sums_route(operand(4, 63, 64), operand(63, 64)) != "torch"
assert host.sums_route(operand(4, 64, address=8), operand(64, 64)) == "torch"
''')
