"""Sizes that run on each form of the products on 4-bit weights: (form, rows, k, n_out, experts), experts = 0 for the plain product.  Rows and
columns end inside a tile, K inside a block, a group of scales or a wave's turn; each form that takes long rows has one of 4096 columns and more."""
CASES = [
    ('raw 8 waves', 1, 1000, 48, 0), ('raw 8 waves', 1, 8191, 4200, 0), ('raw 8 waves', 16, 250, 33, 0),
    ('raw 16 waves', 1, 16384, 200, 0), ('raw 16 waves', 4, 4095, 100, 0), ('raw 16 waves', 15, 1090, 17, 0),
    ('rows 16', 40, 160, 40, 0), ('rows 16', 300, 513, 516, 0), ('rows 16', 77, 1023, 2049, 0), ('rows 16', 5001, 300, 50, 0),
    ('rows 32', 13505, 250, 256, 0), ('rows 32', 24001, 512, 128, 0), ('rows 32', 16000, 2040, 40, 0),
    ('skinny 16 rows 4 waves', 16, 8190, 500, 0), ('skinny 16 rows 4 waves', 7, 4100, 9001, 0),
    ('skinny 16 rows 2 waves', 13, 4097, 17003, 0), ('skinny 16 rows 2 waves', 16, 1040, 16384, 0),
    ('skinny 32 rows 4 waves', 20, 4100, 9001, 0), ('skinny 32 rows 4 waves', 32, 1030, 16384, 0),
    ('skinny 32 rows 8 waves', 64, 4100, 2047, 0), ('skinny 32 rows 8 waves', 301, 16400, 100, 0), ('skinny 32 rows 8 waves', 33, 1025, 2048, 0),
    ('tile 64 x 64', 64, 8200, 2065, 0), ('tile 64 x 64', 301, 1100, 1000, 0), ('tile 64 x 64', 33, 16384, 4104, 0), ('tile 64 x 64', 3000, 2100, 63, 0),
    ('tile 64 x 128', 701, 4100, 4001, 0), ('tile 64 x 128', 513, 8192, 8200, 0), ('tile 64 x 128', 3001, 290, 2008, 0),
    ('tile 128 x 128', 3000, 4100, 2051, 0), ('tile 128 x 128', 4353, 1200, 4104, 0), ('tile 128 x 128', 20001, 2050, 300, 0),
    ('tile 256 x 256', 4090, 4100, 4088, 0), ('tile 256 x 256', 4001, 520, 4090, 0), ('tile 256 x 256', 4096, 8192, 4096, 0),
    ('raw 4 waves', 4, 250, 64, 8), ('raw 4 waves', 16, 1024, 131, 6), ('raw 4 waves', 15, 33, 48, 2),
    ('raw 8 waves', 2, 8190, 48, 8), ('raw 8 waves', 6, 2500, 33, 3),
    ('skinny 16 rows 4 waves', 30, 4100, 200, 40), ('skinny 16 rows 4 waves', 100, 290, 130, 20),
    ('skinny 16 rows 2 waves', 60, 4100, 4090, 60), ('skinny 16 rows 2 waves', 40, 520, 4096, 64),
    ('skinny 32 rows 8 waves', 120, 4100, 208, 5), ('skinny 32 rows 8 waves', 60, 16384, 130, 3),
    ('tile 32 x 128', 128, 4100, 4090, 32), ('tile 32 x 128', 192, 64, 520, 64), ('tile 32 x 128', 900, 300, 4104, 40),
    ('tile 64 x 128', 1800, 64, 520, 64), ('tile 64 x 128', 700, 4100, 4001, 9), ('tile 64 x 128', 1400, 200, 4104, 5),
    ('tile 64 x 64', 300, 4100, 4103, 5), ('tile 64 x 64', 200, 160, 2064, 4),
    ('tile 128 x 128', 6000, 4100, 3001, 3), ('tile 128 x 128', 1900, 160, 9000, 3),
    ('tile 256 x 256', 3900, 4100, 4090, 3), ('tile 256 x 256', 12000, 200, 4096, 4),
]


def form_of(rows, k, n, experts):
    import gunet_amd
    return gunet_amd._lib.lib.gunet_mxfp4_form(rows, k, n, experts).decode()
