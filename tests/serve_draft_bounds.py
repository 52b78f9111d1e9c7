"""The forms of attention over the 16-bit cache, by what chooses them."""

# columns (rows announced x query heads of a KV head) choose the form, and whether the table allows sequences of any length: (rows, query heads a KV head, whether it does, whether weights are rounded once)
FORMS = {"one launch, 8": (1, 4, False, False), "one launch, 16": (3, 5, False, False), "one launch, 32": (5, 4, False, False), "one launch, 64": (9, 7, False, False),
         "a line, 8": (2, 4, True, False), "a line, 16": (3, 5, True, False), "many, boxes": (40, 4, True, True), "many, gathered": (40, 5, True, True)}
