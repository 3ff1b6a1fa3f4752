"""Sizes (rows, channels, hidden, outputs) whose calls reach, between them, every
kernel of the gated feed-forward block's products and joins, and what a call reaches."""
import torch

from riemannengine_amd import abi

SIZES = {
    torch.float32: [
        (4786, 56, 930, 1981), (983, 1106, 2754, 1000), (1364, 3857, 566, 187),
        (1036, 109, 7366, 549), (11195, 12, 1301, 285), (13655, 18, 274, 976),
        (13195, 261, 487, 15), (8135, 1627, 73, 1936), (746, 16, 6599, 590),
        (3090, 93, 2384, 222), (75, 1553, 5175, 2947), (132, 671, 10953, 222),
        (2005, 483, 1005, 41), (4286, 486, 471, 10), (4019, 1489, 68, 3676), (87, 49, 3381, 4071),
        (88, 4027, 1647, 30), (94, 2801, 972, 1533), (2006, 3653, 10, 34), (490, 54, 489, 490),
        (3483, 1686, 8, 1523), (329, 356, 315, 174), (1379, 339, 13, 819)],
    torch.bfloat16: [
        (10176, 9, 6596, 455), (14741, 143, 5969, 12), (13097, 17, 9382, 179),
        (11840, 74, 2294, 71), (5900, 12, 8446, 81), (336, 45, 3562, 3789), (3277, 205, 2310, 42),
        (76, 2174, 6418, 15), (10030, 343, 196, 23), (10608, 1253, 9, 1369), (5474, 2830, 8, 72),
        (1613, 3050, 9, 3673), (17, 2488, 899, 978), (19, 9, 1732, 2334)],
}


def shares(launch):
    """How the tiles of k are divided: a workgroup has each tile, tiles are cut
    evenly, cut anywhere, or stand in a line of which a workgroup has more than one."""
    if launch.parts == 0:
        return "whole"
    if launch.parts % launch.tiles == 0:
        return "even"
    return "uneven" if launch.parts > launch.tiles else "line"


def reached(dtype, sizes):
    """(product, side of a tile, how it is shared, threads of the join) of a call's products."""
    out = set()
    for product in abi.GATED_PRODUCTS:
        launch = abi.gated_plan(product, dtype, *sizes)
        if launch.side:
            out.add((product, launch.side, shares(launch), launch.join))
    return out
