"""Public constants (torchbvh/_constants.py:1-2), with k = 32 added."""

SUPPORTED_K = (4, 8, 16, 32)
SUPPORTED_DIMS = (2, 3)

# Block selection and attention: leaves of a block, most blocks of a query, most
# channels of a head, most buckets of a distance bias.
BLOCK_SIZE = 64
MAX_SELECTED_BLOCKS = 32
MAX_BLOCK_CHANNELS = 128
MAX_BLOCK_HEADS = 4096
MAX_SHARED_HEADS = 64  # query heads of one key/value head
MAX_BIAS_BUCKETS = 64

# Squared distance at or below which a neighbour counts as an exact hit in
# interpolate_displaced, and the inverse-distance weight regulariser
# (torchbvh/_constants.py:3).
EXACT_DISTANCE_EPSILON = 1.0e-12
