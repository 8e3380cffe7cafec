"""For each form of the 4-bit product (mx4_forms.h) rows of X and of W that take it: for every kernel that the library launches a size."""

X4 = {"rows 1x1": (20, 1001), "rows 1x2": (1, 5003), "rows 2x2": (17, 4099), "rows 2x4": (3, 8203), "rows 4x4": (60, 8200), "tile 64x128": (300, 4099),
      "tile 128x128": (300, 8203), "tile 256x128": (520, 8203), "tile 256x256": (1100, 8201)}
X16 = {"rows 1x1 few": (3, 2105), "rows 1x1": (16, 530), "rows 1x2 few": (1, 5003), "rows 1x2": (5, 5120), "rows 1x4 few": (4, 14300), "rows 1x4": (33, 4099),
       "rows 2x4": (60, 4099), "rows 2x4/4": (100, 4099), "tile 64x256": (300, 4099), "tile 128x256": (520, 8203)}
# single tokens and small batches against the widths of a layer's matrices
FEW = [(T, N) for T in (1, 4, 5, 16) for N in (5000, 8200, 14300)]
