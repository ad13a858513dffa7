"""Small programs that use the library as a serving program would."""
